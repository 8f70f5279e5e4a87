"""The gated recurrence and compositing against a plain loop in 64 bits.

Tolerances come with the reference: it carries a bound of the rounding errors along.  With u =
2^-24, a step of the kernel multiplies by a = exp(-g) (off by 4 u, the hardware's power of two, and
1.5 g u, its argument) and by w = 1 - a (below 14 u + u where it is a difference, g >= 0.25; below 3 u
as a series) and adds, in whatever association the stretches are joined; every factor and sum enters
the error once, so with the sums of magnitudes
    H[t] = a H[t-1] + w |x|,   e[t] = a e[t-1] + ((1 + g / 10) a H[t-1] + w |x|)
the state is off by at most 20 u e[t], and likewise the adjoint.  Outputs of 16 bits are rounded once
more, by half a step."""
import pytest
import torch

import svox_b200 as svox
from svox_b200 import csrc

U = 2.0 ** -24
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rows_of(values, offsets):
    if offsets is None:
        n, T = values.shape[:2]
        return [(b * T, b * T + T) for b in range(n)]
    o = offsets.tolist()
    return list(zip(o[:-1], o[1:]))


def reference(values, thickness, initial, offsets, reverse, weighted, d_states=None, d_last=None):
    """Plain loops in 64 bits -> {name: (value, tolerance before the output's rounding)}."""
    C = values.shape[-1]
    x = values.detach().cpu().double().reshape(-1, C)
    g = thickness.detach().cpu().double()
    g = g.reshape(x.shape[0], -1)
    H = g.shape[1]
    D = C // H
    g = g.repeat_interleave(D, 1)
    rows = rows_of(values, None if offsets is None else offsets.cpu())
    B = len(rows)
    h0 = torch.zeros(B, C, dtype=torch.float64) if initial is None else \
        initial.detach().cpu().double().expand(B, C)
    ds = torch.zeros_like(x) if d_states is None else d_states.cpu().double().reshape(-1, C)
    dl = torch.zeros(B, C, dtype=torch.float64) if d_last is None else d_last.cpu().double()
    a = torch.exp(-g)
    w = torch.ones_like(a) if weighted else -torch.expm1(-g)
    f = torch.where(a == 0, torch.ones_like(a), 1 + 0.1 * g)
    take = torch.where(w == 0, torch.zeros_like(x), w * x)
    out = {n: torch.zeros_like(x) for n in ("states", "e_states", "dx", "e_dx", "dgc", "e_dgc")}
    last, e_last, d0, e_d0 = (torch.zeros(B, C, dtype=torch.float64) for _ in range(4))
    for b, (lo, hi) in enumerate(rows):
        steps = list(range(lo, hi))
        if reverse:
            steps.reverse()
        h, Habs, e = h0[b].clone(), h0[b].abs(), torch.zeros(C, dtype=torch.float64)
        before = {}
        for t in steps:
            before[t] = (h, Habs, e)
            gone = a[t] == 0
            z = torch.zeros_like(h)
            ah, aH, ae = (torch.where(gone, z, a[t] * q) for q in (h, Habs, e))
            e = ae + f[t] * aH + take[t].abs()
            h, Habs = ah + take[t], aH + take[t].abs()
            out["states"][t], out["e_states"][t] = h, e
        last[b], e_last[b] = h, e
        G, Gabs, eG = dl[b].clone(), dl[b].abs(), torch.zeros(C, dtype=torch.float64)
        for t in reversed(steps):
            G, Gabs = G + ds[t], Gabs + ds[t].abs()
            eG = eG + Gabs
            out["dx"][t], out["e_dx"][t] = w[t] * G, w[t] * (eG + Gabs)
            hp, Hp, ep = before[t]
            xt = torch.where((w[t] == 0) & ~x[t].isfinite(), hp, x[t])
            gone = a[t] == 0
            z = torch.zeros_like(h)
            q = torch.where(gone, z, a[t] * (-hp if weighted else xt - hp))
            qa = torch.where(gone, z, a[t] * (Hp if weighted else xt.abs() + Hp))
            qe = torch.where(gone, z, a[t] * ep)
            out["dgc"][t] = q * G
            out["e_dgc"][t] = qa * (eG + f[t] * Gabs) + qe * Gabs + D * qa * Gabs / 20
            G, Gabs, eG = (torch.where(gone, z, a[t] * v) for v in (G, Gabs, eG + f[t] * Gabs))
        d0[b], e_d0[b] = G, eG

    def grouped(v):
        return v.reshape(-1, H, D).sum(2).reshape(thickness.shape)

    shape = values.shape
    tol = 20 * U
    return {"states": (out["states"].reshape(shape), tol * out["e_states"].reshape(shape)),
            "last": (last, tol * e_last), "d_initial": (d0, tol * e_d0),
            "d_values": (out["dx"].reshape(shape), tol * out["e_dx"].reshape(shape)),
            "d_thickness": (grouped(out["dgc"]), tol * grouped(out["e_dgc"]))}


def close(name, got, want):
    value, tol = want
    assert got.shape == value.shape, name
    g = got.detach().cpu().double()
    # (what is below 2^-149 in 32 bits is 0: an error of at most that much in each of the fewer than
    # 2^20 products that an output here consists of, times other factors below 2^20)
    tol = tol + HALF_STEP[got.dtype] * (value.abs() + tol) + 2.0 ** -109
    if got.dtype == F16:
        tol = tol + 2.0 ** -25          # half of its smallest step
    off = (g - value).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (name, int(bad.sum()), off[bad].max().item(),
                           bad.nonzero()[0].tolist())


def inputs(gen, lead, C, H, dtype, gates, dev):
    x = torch.randn(*lead, C, generator=gen).to(dev, dtype)
    g = torch.exp(1.5 * torch.randn(*lead, *([H] if H > 1 else []), generator=gen) - 2)
    g[torch.rand(g.shape, generator=gen) < 0.2] = 0.0
    g[torch.rand(g.shape, generator=gen) < 0.05] = 12.0
    return x, g.to(dev, gates)


def check_call(dev, x, g, initial, offsets, reverse, weighted, gen, with_states=True,
               with_last=True):
    for t in (x, g, initial):
        if t is not None:
            t.requires_grad_(True)
    states, last = svox.gated_scan(x, g, initial, offsets, reverse, weighted)
    assert states.dtype == x.dtype and last.dtype == F32
    ds = torch.randn(states.shape, generator=gen).to(dev, states.dtype) if with_states else None
    dl = torch.randn(last.shape, generator=gen).to(dev) if with_last else None
    want = reference(x, g, initial, offsets, reverse, weighted, ds, dl)
    close("states", states, want["states"])
    close("last", last, want["last"])
    outs = [o for o, d in ((states, ds), (last, dl)) if d is not None]
    leaves = [t for t in (x, g, initial) if t is not None]
    grads = torch.autograd.grad(outs, leaves, [d for d in (ds, dl) if d is not None])
    close("d_values", grads[0], want["d_values"])
    close("d_thickness", grads[1], want["d_thickness"])
    if initial is not None and initial.shape == last.shape:
        close("d_initial", grads[2], want["d_initial"])
    with torch.no_grad():       # the call that keeps nothing
        again = svox.gated_scan(x, g, initial, offsets, reverse, weighted)
    assert torch.equal(again[0], states) and torch.equal(again[1], last)
    return states, last, grads


# (B, T, C, H): one step to several stretches and splits, odd sizes, gates of all kinds
SHAPES = [(2, 300, 128, 2), (1, 700, 128, 8), (1, 3000, 128, 2), (170, 20, 64, 64),
          (3, 150, 6, 2), (2, 200, 128, 128), (1, 3000, 64, 64), (1, 1, 1, 1), (3, 1, 5, 5), (2, 2, 3, 1), (2, 63, 33, 33), (1, 64, 64, 64), (3, 65, 66, 66),
          (2, 130, 7, 7), (1, 257, 48, 3), (2, 71, 96, 4), (1, 40, 200, 1), (2, 33, 130, 2),
          (5, 19, 34, 17), (1, 1500, 3, 1), (1, 1029, 70, 70), (40, 9, 16, 16), (2, 700, 1, 1),
          (3, 100, 12, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype,gates", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16),
                                         (F16, F32)])
def test_scan(cuda_device, shape, dtype, gates):
    B, T, C, H = shape
    gen = torch.Generator().manual_seed(B + T + C)
    for k, (reverse, weighted) in enumerate([(False, False), (True, True)]):
        x, g = inputs(gen, (B, T), C, H, dtype, gates, cuda_device)
        initial = torch.randn(B, C, generator=gen).to(cuda_device) if k == 0 or T > 50 else None
        check_call(cuda_device, x, g, initial, None, reverse, weighted, gen)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("C,H,dtype", [(3, 1, F32), (1, 1, F32), (4, 4, F16), (40, 8, BF16),
                                       (66, 66, BF16), (33, 1, F32), (3, 1, BF16), (16, 1, F32),
                                       (6, 2, F32), (130, 1, F32)])
def test_packed(cuda_device, C, H, dtype, reverse):
    """Rows of any length, empty ones among them, and steps that no row covers."""
    gen = torch.Generator().manual_seed(C)
    n = torch.tensor([0, 1, 5, 0, 0, 130, 64, 65, 2, 300, 0, 31, 32, 33, 0])
    offsets = (7 + torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)])).to(cuda_device)
    N = int(offsets[-1]) + 11
    x, g = inputs(gen, (N,), C, H, dtype, F32, cuda_device)
    initial = torch.randn(n.numel(), C, generator=gen).to(cuda_device)
    # the outputs' memory is not clean
    junk = [torch.full((N * max(C, 64),), float("nan"), device=cuda_device) for _ in range(4)]
    del junk
    states, last, grads = check_call(cuda_device, x, g, initial, offsets, reverse, False, gen)
    for t in (states, grads[0], grads[1]):
        assert (t[:7] == 0).all() and (t[-11:] == 0).all()
    empty = (n == 0).to(cuda_device)
    assert torch.equal(last[empty], initial[empty])
    assert csrc.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("C,dtype", [(1, F32), (2, F32), (3, F32), (3, BF16), (4, F32), (7, F16),
                                     (8, BF16), (32, BF16), (35, F32), (64, F16), (5, BF16),
                                     (12, F32), (100, F32), (128, BF16), (200, F32), (77, F16),
                                     (128, F32), (127, F32)])
@pytest.mark.parametrize("packed", [True, False])
def test_composite(cuda_device, C, dtype, packed):
    gen = torch.Generator().manual_seed(C)
    if packed:
        n = torch.cat([torch.randint(0, 70, (60,), generator=gen), torch.tensor([0, 0, 900, 1, 0])])
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(cuda_device)
        lead, B = (int(offsets[-1]),), n.numel()
    else:
        offsets, lead, B = None, (37, 45), 37
    x, g = inputs(gen, lead, C, 1, dtype, F32, cuda_device)
    bg = torch.rand(B, C, generator=gen).to(cuda_device)
    for t in (x, g, bg):
        t.requires_grad_(True)
    out = svox.composite(x, g, bg, offsets)
    d = torch.randn(out.shape, generator=gen).to(cuda_device)
    want = reference(x, g, bg, offsets, True, False, None, d)
    close("last", out, want["last"])
    for name, got in zip(("d_values", "d_thickness", "d_initial"),
                         torch.autograd.grad([out], [x, g, bg], [d])):
        close(name, got, want[name])
    close("last", svox.gated_scan(x, g, bg, offsets, reverse=True)[1], want["last"])
    with torch.no_grad():
        assert torch.equal(out, svox.composite(x, g, bg, offsets))


@pytest.mark.gpu
@pytest.mark.parametrize("B,mean", [(200_000, 5), (130_000, 40), (60_000, 80), (130_000, 0)])
def test_many_rays(cuda_device, B, mean):
    """So many rays that a warp orders a number of them by length; `mean` 0: 37 samples each.

    Weights are at most 1 together and values at most 1.  A weight is off by 30 u (see above) and
    what reaches it, T, a product of i factors that are off by 4 u each and rounded once, by 5 i T u; a
    gradient by as much times |d|, twice."""
    gen = torch.Generator(device=cuda_device).manual_seed(B)
    if mean:
        n = (torch.empty(B, device=cuda_device).exponential_(1 / mean, generator=gen)).long()
        n[torch.rand(B, device=cuda_device, generator=gen) < 0.2] = 0
        offsets = torch.cat([n.new_zeros(1), n.cumsum(0)])
        N = int(offsets[-1])
    else:
        N = B * 37
        offsets = torch.arange(B + 1, device=cuda_device) * 37
        n = offsets.diff()
    x = torch.rand(N, 3, device=cuda_device, generator=gen)
    g = torch.rand(N, device=cuda_device, generator=gen) ** 4 * 2
    bg = torch.rand(B, 3, device=cuda_device, generator=gen)
    d = torch.randn(B, 3, device=cuda_device, generator=gen)
    leaves = [t.requires_grad_(True) for t in (x, g, bg)]
    if mean:
        out = svox.composite(*leaves, offsets)
    else:
        out = svox.composite(x.view(B, 37, 3), g.view(B, 37), bg)
    got = torch.autograd.grad(out, leaves, d)
    with torch.no_grad():
        ray = torch.repeat_interleave(torch.arange(B, device=cuda_device), n)
        upto = torch.cat([g.new_zeros(1).double(), g.double().cumsum(0)])
        T = torch.exp(upto[offsets[:-1]][ray] - upto[:-1])
        end = torch.exp(upto[offsets[:-1]] - upto[offsets[1:]])
        w = T * -torch.expm1(-g.double())
        total = torch.zeros(B, 3, dtype=torch.float64, device=cuda_device)
        total.index_add_(0, ray, w[:, None] * x)
        i = torch.arange(N, device=cuda_device) - offsets[:-1][ray]
        tol = (30 + 5 * float((i * T).max()) + 5 * float((n * end).max())) * U
        assert (out - (total + end[:, None] * bg)).abs().max() <= tol + U
        c = (d.double()[ray] * x).sum(1)
        wc = torch.cat([w.new_zeros(1), (w * c).cumsum(0)])
        behind = wc[offsets[1:]][ray] - wc[1:] + (end * (d * bg).sum(1))[ray]
        size = d.abs().sum(1).double()
        assert ((got[0] - w[:, None] * d[ray]).abs() <= (tol + U) * d.abs()[ray]).all()
        assert ((got[1] - (T * torch.exp(-g.double()) * c - behind)).abs() <=
                2 * (tol + 3 * U) * size[ray] + N * 2.0 ** -52 * size.max()).all()
        assert ((got[2] - end[:, None] * d).abs() <= (tol + U) * d.abs()).all()


@pytest.mark.gpu
def test_composite_is_emission_and_absorption(cuda_device):
    """The sum of what each sample emits, weighted by what reaches it."""
    gen = torch.Generator().manual_seed(0)
    x, g = inputs(gen, (50, 90), 3, 1, F32, F32, cuda_device)
    bg = torch.rand(3, generator=gen).to(cuda_device)
    through = torch.exp(-(g.double().cumsum(1) - g.double()))
    w = through * -torch.expm1(-g.double())
    want = (w[..., None] * x).sum(1) + torch.exp(-g.double().sum(1))[:, None] * bg
    tol = reference(x, g, bg, None, True, False)["last"][1]
    close("last", svox.composite(x, g, bg), (want.cpu(), tol))


@pytest.mark.gpu
def test_gradients_against_differences(cuda_device):
    """Central differences of the kernel's own output.  Their truncation error is the reference's,
    found in 64 bits; the kernel's rounding is divided by the step."""
    gen = torch.Generator().manual_seed(3)
    x, g = inputs(gen, (4, 40), 3, 1, F32, F32, cuda_device)
    bg = torch.rand(4, 3, generator=gen).to(cuda_device)
    g = g.clamp(min=0.05)
    d = torch.randn(4, 3, generator=gen).to(cuda_device)
    step = 2.0 ** -6
    leaves = [t.clone().requires_grad_(True) for t in (x, g, bg)]
    grads = torch.autograd.grad([svox.composite(*leaves)], leaves, [d])

    def plain(x, g, bg):
        want = reference(x, g, bg, None, True, False)["last"]
        return (want[0] * d.cpu()).sum().item(), (want[1] * d.cpu().abs()).sum().item()

    for k in range(3):
        way = torch.randn(leaves[k].shape, generator=gen).to(cuda_device)
        way = (way * 16).round() / 16
        ends = []
        for sign in (1, -1):
            args = [x, g, bg]
            args[k] = args[k] + sign * step * way
            ends.append(([(svox.composite(*args).double() * d).sum().item()], plain(*args)))
        slope = (ends[0][0][0] - ends[1][0][0]) / (2 * step)
        exact = (ends[0][1][0] - ends[1][1][0]) / (2 * step)
        want = reference(x, g, bg, None, True, False, None, d)
        name = ("d_values", "d_thickness", "d_initial")[k]
        along = (want[name][0] * way.cpu()).sum().item()
        mine = (grads[k].double() * way).sum().item()
        rounding = (ends[0][1][1] + ends[1][1][1]) / (2 * step) + \
            (want[name][1] * way.cpu().abs()).sum().item()
        assert abs(mine - slope) <= abs(exact - along) + rounding


@pytest.mark.gpu
def test_strides_and_broadcasts(cuda_device):
    """Slices of a wider projection, broken alignment, transposed and expanded inputs, a state for
    all rows: the same results as their copies, and gradients of the right shape."""
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(3, 70, 150, generator=gen).to(cuda_device)
    gate = torch.rand(3, 70, 150, generator=gen).to(cuda_device)
    flat = torch.randn(3 * 70 * 64 + 1, generator=gen).to(cuda_device, BF16)
    cases = [(wide[:, :, 5:69], gate[:, :, 3:67]), (wide[:, :, 4:68], gate[:, :, 2:66]),
             (wide[:, ::2, 4:68], gate[:, ::2, 2:66]), (wide[1:, :, 1:4], gate[1:, :, 7]),
             (wide.transpose(1, 2)[:, 3:40, :], gate.transpose(1, 2)[:, 3:40, :]),
             (wide[:, :1, 4:68].expand(3, 70, 64), gate[:1, :, 0].expand(3, 70)),
             (flat[1:].view(3, 70, 64), gate[:, :, 9:73].to(BF16)),
             (wide[:, :, 4:5], gate[:, :, 4:5])]
    for x, g in cases:
        state = torch.randn(x.shape[-1], generator=gen).to(cuda_device)
        a = [x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True),
             g.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True),
             state.clone().requires_grad_(True)]
        b = [x.detach().requires_grad_(True), g.detach().requires_grad_(True),
             state.clone().requires_grad_(True)]
        outs = [svox.gated_scan(*v[:2], initial=v[2]) for v in (a, b)]
        d = [torch.randn(o.shape, generator=gen).to(cuda_device, o.dtype) for o in outs[0]]
        for p, q in zip(outs[0], outs[1]):
            assert torch.equal(p, q)
        for p, q in zip(torch.autograd.grad(outs[0], a, d), torch.autograd.grad(outs[1], b, d)):
            assert p.shape == q.shape and torch.equal(p, q)
        want = reference(x, g, state, None, False, False, d[0], d[1])
        close("states", outs[1][0], want["states"])
        # one state for all rows: its gradient is summed over them (a rounding for each)
        total = want["d_initial"][0].sum(0), want["d_initial"][1].sum(0) + \
            want["d_initial"][0].abs().sum(0) * 3 * U
        states, last = svox.gated_scan(*b[:2], initial=b[2])
        close("d_initial", torch.autograd.grad([states, last], b[2], d)[0], total)
    # an unaligned gradient
    x = torch.randn(2, 30, 64, generator=gen).to(cuda_device, BF16).requires_grad_(True)
    g = torch.rand(2, 30, 64, generator=gen).to(cuda_device, BF16)
    states, last = svox.gated_scan(x, g)
    d = torch.randn(2 * 30 * 64 + 1, generator=gen).to(cuda_device, BF16)[1:].view(2, 30, 64)
    assert d.data_ptr() % 4 == 2
    close("d_values", torch.autograd.grad(states, x, d)[0],
          reference(x, g, None, None, False, False, d)["d_values"])


@pytest.mark.gpu
@pytest.mark.parametrize("C", [1, 2, 3, 4])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_composite_wherever_it_lies(cuda_device, C, dtype):
    """Rays of every length at every place of a quad, in an array that ends anywhere; values and
    gradients off their boundaries, and with strides."""
    gen = torch.Generator().manual_seed(C)
    for lengths in (list(range(1, 40)) + [0, 0, 127, 128, 129, 3, 1], [5], [4], [1, 1, 1], [0, 2, 0],
                    [600] * 5, [2500, 3, 0, 2499]):
        n = torch.tensor(lengths)
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(cuda_device)
        N = int(n.sum())
        x, g = inputs(gen, (N,), C, 1, dtype, F32 if C % 2 else dtype, cuda_device)
        bg = torch.rand(n.numel(), C, generator=gen).to(cuda_device)
        d = torch.randn(n.numel(), C, generator=gen).to(cuda_device)
        want = reference(x, g, bg, offsets, True, False, None, d)
        flat = torch.zeros(N * C + 1, device=cuda_device, dtype=dtype)
        flat[1:] = x.flatten()
        wide = torch.zeros(N, C + 2, device=cuda_device, dtype=dtype)
        wide[:, 1:-1] = x
        gates = torch.zeros(N, 2, device=cuda_device, dtype=g.dtype)
        gates[:, 1] = g
        for xv, gv in ((x, g), (flat[1:].view(N, C), g), (wide[:, 1:-1], g), (x, gates[:, 1])):
            leaves = [xv.detach().requires_grad_(True), gv.detach().requires_grad_(True),
                      bg.clone().requires_grad_(True)]
            out = svox.composite(*leaves, offsets)
            close("last", out, want["last"])
            for name, got in zip(("d_values", "d_thickness", "d_initial"),
                                 torch.autograd.grad(out, leaves, d)):
                close(name, got, want[name])
            with torch.no_grad():
                assert torch.equal(svox.composite(xv, gv, bg, offsets), out)
    for premultiplied in (False, True):
        x, g = inputs(gen, (3, 37), C, 1, dtype, F32, cuda_device)
        x.requires_grad_(True)
        g.requires_grad_(True)
        out = svox.composite(x, g, premultiplied=premultiplied)
        d = torch.randn(3, C, generator=gen).to(cuda_device)
        want = reference(x, g, None, None, True, premultiplied, None, d)
        close("last", out, want["last"])
        grads = torch.autograd.grad(out, [x, g], d)
        close("d_values", grads[0], want["d_values"])
        close("d_thickness", grads[1], want["d_thickness"])


@pytest.mark.gpu
@pytest.mark.parametrize("C,H,T", [(64, 4, 1500), (64, 64, 1500), (6, 2, 90), (3, 3, 40), (32, 1, 70),
                                   (300, 1, 50), (37, 1, 70), (200, 1, 1500)])
@pytest.mark.parametrize("premultiplied", [False, True])
def test_composite_groups(cuda_device, C, H, T, premultiplied):
    """Thickness of groups of channels or of each, and values weighted beforehand; long rays."""
    gen = torch.Generator().manual_seed(C + H)
    x, g = inputs(gen, (2, T), C, H, BF16, F32, cuda_device)
    bg = torch.rand(C, generator=gen).to(cuda_device)
    with torch.no_grad():
        alone = svox.composite(x, g, bg, premultiplied=premultiplied)
    leaves = [t.requires_grad_(True) for t in (x, g)]
    out = svox.composite(x, g, bg, premultiplied=premultiplied)
    d = torch.randn(out.shape, generator=gen).to(cuda_device)
    want = reference(x, g, bg, None, True, premultiplied, None, d)
    close("last", out, want["last"])
    close("last", alone, want["last"])
    for name, got in zip(("d_values", "d_thickness"), torch.autograd.grad(out, leaves, d)):
        close(name, got, want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("C", [3, 64])
def test_masked_places(cuda_device, C):
    """Samples of no thickness may hold anything; nothing from behind an opaque sample shows."""
    gen = torch.Generator().manual_seed(2)
    x, g = inputs(gen, (6, 150), C, 1, F32, F32, cuda_device)
    bg = torch.rand(6, C, generator=gen).to(cuda_device)
    masked = torch.rand(6, 150, generator=gen).to(cuda_device) < 0.3
    masked[5] = True                                   # a row whose mask leaves nothing
    g = torch.where(masked, torch.zeros_like(g), g)
    dirty = torch.where(masked[..., None], torch.full_like(x, float("nan")), x)
    dirty[0][masked[0]] = float("inf")
    dirty[1][masked[1]] = torch.finfo(F32).min
    clean = torch.where(masked[..., None], torch.zeros_like(x), x)
    d = torch.randn(6, C, generator=gen).to(cuda_device)
    got = []
    for v in (clean, dirty):
        leaves = [v.clone().requires_grad_(True), g.clone().requires_grad_(True),
                  bg.clone().requires_grad_(True)]
        out = svox.composite(*leaves)
        got.append([out, *torch.autograd.grad(out, leaves, d)])
    assert torch.equal(got[0][0], got[1][0])
    assert torch.equal(got[0][0][5], bg[5])
    assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][3], got[1][3])
    assert torch.equal(got[0][2][~masked], got[1][2][~masked])
    # (row 1 holds the lowest float where it is masked: with no thickness the gradient is its true sum
    # over the channels, up to 64 times 3.4e38 times the adjoint, which is beyond the largest float)
    rest = [0, 2, 3, 4, 5]
    assert got[1][2][rest].isfinite().all()
    # opaque: thickness inf, and what is behind it is not a number
    g[:, 40] = float("inf")
    dirty = clean.clone()
    dirty[:, 41:] = float("nan")
    bg[:] = float("nan")
    g[:, 41:] = g[:, 41:].clamp(min=0.1)
    leaves = [dirty.requires_grad_(True), g.requires_grad_(True), bg.requires_grad_(True)]
    out = svox.composite(*leaves)
    want = reference(clean[:, :41], g[:, :41], None, None, True, False, None, d)
    close("last", out, want["last"])
    grads = torch.autograd.grad(out, leaves, d)
    close("d_values", grads[0][:, :41], want["d_values"])
    assert (grads[0][:, 41:] == 0).all() and (grads[2] == 0).all()
    assert grads[1][:, :41].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("C", [1, 3, 32, 64, 300])
@pytest.mark.parametrize("premultiplied", [False, True])
def test_behind_an_opaque_sample(cuda_device, C, premultiplied):
    """Nothing of what is behind it counts, a thickness that is not a number neither: not for what is
    seen, and not for the gradients of what is in front."""
    gen = torch.Generator().manual_seed(C)
    x, g = inputs(gen, (5, 90), C, 1, F32, F32, cuda_device)
    at = [0, 1, 37, 70, 88]
    for row, k in enumerate(at):
        g[row, k] = float("inf")
        g[row, k + 1:] = float("nan")
        x[row, k + 1:] = float("nan")
    bg = torch.full((5, C), float("nan"), device=cuda_device)
    d = torch.randn(5, C, generator=gen).to(cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, g, bg)]
    for xv, gv, offsets in ((x, g, None), (x.view(-1, C), g.view(-1),
                                           torch.arange(6, device=cuda_device) * 90)):
        out = svox.composite(xv, gv, bg, offsets, premultiplied)
        grads = torch.autograd.grad(out, leaves, d)
        for row, k in enumerate(at):
            part = slice(row, row + 1), slice(0, k + 1)
            want = reference(x[part], g[part], None, None, True, premultiplied, None, d[part[0]])
            close("last", out[part[0]], want["last"])
            close("d_values", grads[0][part], want["d_values"])
            close("d_thickness", grads[1][part], want["d_thickness"])
    # in front of it, it counts
    with torch.no_grad():
        g[2, 5] = float("nan")
        assert svox.composite(x, g, bg)[2].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,C,H", [(3, 90, 6, 1), (3, 90, 6, 3), (2, 700, 70, 70), (1, 6000, 64, 64),
                                     (1, 6000, 64, 2), (1, 6000, 5, 1), (2, 5, 8, 1)])
@pytest.mark.parametrize("premultiplied", [False, True])
def test_states_past_an_opaque_step(cuda_device, B, T, C, H, premultiplied):
    """Whatever the thickness before it, NaN too: from the opaque step on, all states are those of a row
    that begins there, in rows of several ranges as well."""
    gen = torch.Generator().manual_seed(T + C)
    x, g = inputs(gen, (B, T), C, H, F32, F32, cuda_device)
    k = T * 2 // 3
    g[:, k] = float("inf")
    g[:, 1:k] = float("nan")
    h0 = torch.full((B, C), float("nan"), device=cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, g, h0)]
    states, last = svox.gated_scan(x, g, h0, premultiplied=premultiplied)
    d_states = torch.randn(states.shape, generator=gen).to(cuda_device)
    d_last = torch.randn(last.shape, generator=gen).to(cuda_device)
    grads = torch.autograd.grad((states, last), leaves, (d_states, d_last))
    part = slice(None), slice(k, None)
    want = reference(x[part], g[part], None, None, False, premultiplied, d_states[part], d_last)
    close("states", states[part], want["states"])
    close("last", last, want["last"])
    close("d_values", grads[0][part], want["d_values"])
    close("d_thickness", grads[1][part], want["d_thickness"])
    assert states[:, 1:k].isnan().all()


@pytest.mark.gpu
def test_partial_gradients(cuda_device):
    """Only some outputs used, only some inputs asked for."""
    gen = torch.Generator().manual_seed(4)
    # (1500 and 2100 steps: ranges of a row in several blocks)
    for C, H, T in ((66, 66, 90), (3, 1, 90), (96, 2, 90), (64, 64, 1500), (128, 128, 2100),
                    (64, 1, 1500), (7, 1, 1500)):
        x, g = inputs(gen, (2, T), C, H, F32, F32, cuda_device)
        s0 = torch.randn(2, C, generator=gen).to(cuda_device)
        check_call(cuda_device, x, g, s0, None, False, False, gen, with_last=False)
        check_call(cuda_device, x.detach(), g.detach(), s0.detach(), None, True, False, gen,
                   with_states=False)
        d = torch.randn(2, C, generator=gen).to(cuda_device)
        args = [x.detach(), g.detach(), s0.detach()]
        for k in range(3):
            v = [t.clone() for t in args]
            v[k].requires_grad_(True)
            want = reference(*args, None, True, False, None, d)
            got, = torch.autograd.grad(svox.composite(*v), [v[k]], d)
            close(k, got, want[("d_values", "d_thickness", "d_initial")[k]])


@pytest.mark.gpu
def test_steps_carry_on(cuda_device):
    """A sequence run in pieces, the last of single steps."""
    gen = torch.Generator().manual_seed(5)
    x, g = inputs(gen, (3, 100), 70, 70, F32, F32, cuda_device)
    want = reference(x, g, None, None, False, False)
    states, state = [], None
    for lo, hi in [(0, 40), (40, 80)] + [(t, t + 1) for t in range(80, 100)]:
        s, state = svox.gated_scan(x[:, lo:hi], g[:, lo:hi], state)
        states.append(s)
    close("states", torch.cat(states, 1), want["states"])
    close("last", state, want["last"])


@pytest.mark.gpu
def test_empty(cuda_device):
    z = torch.zeros
    for lead in ((0, 5), (4, 0), (0, 0)):
        x = z(*lead, 3, device=cuda_device, requires_grad=True)
        g = z(*lead, device=cuda_device, requires_grad=True)
        s0 = torch.rand(lead[0], 3, device=cuda_device).requires_grad_(True)
        states, last = svox.gated_scan(x, g, s0)
        assert states.shape == x.shape and torch.equal(last, s0)
        (states.sum() + last.sum()).backward()
        assert x.grad.shape == x.shape and g.grad.shape == g.shape
        assert torch.equal(s0.grad, torch.ones_like(s0))
    none = z(1, dtype=torch.int64, device=cuda_device)
    x = torch.rand(4, 3, device=cuda_device).requires_grad_(True)
    g = torch.rand(4, device=cuda_device).requires_grad_(True)
    states, last = svox.gated_scan(x, g, offsets=none)
    assert last.shape == (0, 3) and (states == 0).all()
    states.sum().backward()
    assert (x.grad == 0).all() and (g.grad == 0).all()
    rays = z(6, dtype=torch.int64, device=cuda_device)
    x, g = z(0, 3, device=cuda_device), z(0, device=cuda_device)
    bg = torch.rand(3, device=cuda_device)
    assert torch.equal(svox.composite(x, g, bg, rays), bg.expand(5, 3))
    csrc.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("C,H", [(3, 1), (32, 1), (64, 64), (66, 2)])
def test_buffers_that_are_not_full(cuda_device, C, H):
    """Far more room than samples (a buffer of fixed size): zeros in all of it, whatever lies there."""
    gen = torch.Generator().manual_seed(9)
    offsets = torch.tensor([4001, 4041, 4041, 4100], device=cuda_device)
    N = 300_000
    x = torch.full((N, C), float("nan"), device=cuda_device)
    g = torch.full((N, H) if H > 1 else (N,), float("nan"), device=cuda_device)
    some, gates = inputs(gen, (99,), C, H, F32, F32, cuda_device)
    x[4001:4100], g[4001:4100] = some, gates
    x.requires_grad_(True)
    g.requires_grad_(True)
    junk = [torch.full((N * C,), float("nan"), device=cuda_device) for _ in range(4)]
    del junk
    states, last = svox.gated_scan(x, g, offsets=offsets, reverse=True)
    d = torch.randn(3, C, generator=gen).to(cuda_device)
    want = reference(some, gates, None, offsets - 4001, True, False, None, d)
    close("states", states[4001:4100], want["states"])
    grads = [torch.autograd.grad(last, [x, g], d)]
    if H == 1:
        grads.append(torch.autograd.grad(svox.composite(x, g, offsets=offsets), [x, g], d))
    for t in (states, *[t for pair in grads for t in pair]):
        assert (t[:4001] == 0).all() and (t[4100:] == 0).all()
    for dx, dg in grads:
        close("d_values", dx[4001:4100], want["d_values"])
        close("d_thickness", dg[4001:4100], want["d_thickness"])
    assert csrc.device_status() == 0


@pytest.mark.gpu
def test_repeatable_streams_and_graphs(cuda_device):
    gen = torch.Generator().manual_seed(6)
    for lead, C, H, offsets in (((2, 900), 96, 1, None), ((1, 5000), 40, 40, None),
                                ((2000,), 3, 1, torch.tensor([0, 700, 700, 2000]))):
        x, g = inputs(gen, lead, C, H, F32, F32, cuda_device)
        offsets = None if offsets is None else offsets.to(cuda_device)
        x.requires_grad_(True)
        g.requires_grad_(True)

        def step():
            # (no graph of the leaves outlives a step: their accumulation nodes would tie the
            # capture to the stream that they were made on)
            states, last = svox.gated_scan(x, g, offsets=offsets)
            grads = torch.autograd.grad([states.sum() + last.sum()], [x, g])
            return [states.detach(), last.detach(), *grads]

        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                got = step()
        torch.cuda.current_stream().wait_stream(side)
        for p, q in zip(want, got):
            assert torch.equal(p, q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        with torch.no_grad():
            x += 0.25
            for t in held:
                t.fill_(float("nan"))
        for _ in range(2):
            graph.replay()
        for p, q in zip(step(), held):
            assert torch.equal(p, q)


@pytest.mark.gpu
def test_long_axis_past_32_bits(cuda_device):
    """More than 2^31 elements: the last steps, behind one that forgets all before it."""
    T, C = (1 << 21) + 5, 1030
    x = torch.ones(1, T, C, dtype=BF16, device=cuda_device)
    g = torch.full((1, T), 0.5, device=cuda_device)
    assert x.numel() > 1 << 31
    gen = torch.Generator().manual_seed(7)
    tail = torch.randn(1, 20, C, generator=gen).to(cuda_device, BF16)
    x[:, -20:] = tail
    g[:, -20] = float("inf")
    states, last = svox.gated_scan(x, g)
    want = reference(tail, g[:, -20:], None, None, False, False)
    close("states", states[:, -20:], want["states"])
    close("last", last, want["last"])
    del states
    out = svox.composite(x[:, -20:], g[:, -20:])
    g[:, -20] = 0.5
    g[:, 3] = float("inf")
    head = reference(x[:, :4], g[:, :4], None, None, True, False)
    close("last", svox.composite(x, g), head["last"])
    assert out.shape == last.shape


@pytest.mark.gpu
def test_bad_offsets_are_noticed(cuda_device):
    x = torch.rand(50, 3, device=cuda_device).requires_grad_(True)
    g = torch.rand(50, device=cuda_device).requires_grad_(True)
    for bad in ([0, 30, 20, 50], [0, 10, 60], [-5, 10, 50], [0, 1 << 40, 50], [70, 80, 90]):
        csrc.device_status()
        o = torch.tensor(bad, device=cuda_device)
        states, last = svox.gated_scan(x, g, offsets=o)
        (states.sum() + last.sum()).backward()
        svox.composite(x, g, offsets=o).sum().backward()
        assert csrc.device_status() == 9
        assert csrc.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("C", [3, 32, 200])
def test_saved_tensors_elsewhere(cuda_device, C):
    """A backward pass run twice, and one whose saved tensors lie elsewhere than the forward's: off
    their boundaries and back on them."""
    gen = torch.Generator().manual_seed(8)
    n = torch.tensor([30, 0, 77, 5, 1])
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(cuda_device)
    N = int(n.sum())
    flat = torch.randn(N * C + 1, generator=gen).to(cuda_device)
    gates = torch.rand(N + 1, generator=gen).to(cuda_device)
    d = torch.randn(5, C, generator=gen).to(cuda_device)

    def off(t):         # the same values, four bytes off a boundary
        to = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        to[1:] = t.flatten()
        return to[1:].view(t.shape)

    def run(x, g, pack=None, unpack=None):
        x, g = x.detach().requires_grad_(True), g.detach().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(pack or (lambda t: t),
                                                      unpack or (lambda t: t)):
            out = svox.composite(x, g, offsets=offsets)
        first = torch.autograd.grad(out, [x, g], d, retain_graph=True)
        again = torch.autograd.grad(out, [x, g], d)
        for p, q in zip(first, again):
            assert torch.equal(p, q)
        return [out.detach(), *first]

    here, there = (flat[:-1].view(N, C), gates[:-1]), (flat[1:].view(N, C), gates[1:])
    for x, g in (here, there):
        ref = reference(x, g, None, offsets, True, False, None, d)
        # (other addresses may mean another order of a sum over channels)
        for hooks in ((None, None), (None, lambda t: off(t) if t.dtype == F32 else t),
                      (None, lambda t: t.clone()), (lambda t: t.cpu(), lambda t: t.to(cuda_device))):
            out = run(x, g, *hooks)
            for name, got in zip(("last", "d_values", "d_thickness"), out):
                close(name, got, ref[name])


@pytest.mark.gpu
def test_no_second_derivative_and_edits(cuda_device):
    x = torch.rand(2, 30, 3, device=cuda_device, requires_grad=True)
    g = torch.rand(2, 30, device=cuda_device, requires_grad=True)
    grads = torch.autograd.grad(svox.composite(x, g).sum(), [x, g], create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        grads[0].sum().backward()
    out = svox.composite(x, g)
    with torch.no_grad():
        x += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        dual = fwad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            svox.composite(dual, g.detach())


def test_refusals():
    x, g = torch.rand(2, 5, 6), torch.rand(2, 5)
    o = torch.tensor([0, 3, 5])
    bad = [((x.double(), g), {}, "float32, bfloat16 or float16"),
           ((x[0], g), {}, r"\(B, T, C\)"), ((x, g), {"offsets": o}, r"\(N, C\)"),
           ((x[..., :0], g), {}, "must have a channel"),
           ((x, g[:, :4]), {}, "the steps of values"), ((x, g[0]), {}, "thickness must be"),
           ((x, g.bfloat16()), {}, "float32 or of the type"),
           ((x.bfloat16(), g.half()), {}, "float32 or of the type"),
           ((x, torch.rand(2, 5, 4)), {}, "multiple"), ((x, torch.rand(2, 5, 0)), {}, "multiple"),
           ((x[0], g[0]), {"offsets": o.int()}, "int64"),
           ((x[0], g[0]), {"offsets": o[None]}, "int64"),
           ((x[0], g[0]), {"offsets": o[:0]}, "int64"),
           ((x, g), {"initial": torch.rand(3, 6)}, "initial must be"),
           ((x, g), {"initial": torch.rand(2, 4)}, "initial must be"),
           ((x, g), {"initial": torch.rand(1, 2, 6)}, "initial must be"),
           ((x, g), {"initial": torch.ones(2, 6, dtype=torch.int64)}, "floating"),
           ((x, g), {}, "CUDA tensor"), ((x[0], g[0]), {"offsets": o}, "CUDA tensor")]
    for args, more, text in bad:
        with pytest.raises(RuntimeError, match=text):
            svox.gated_scan(*args, **more)
    with pytest.raises(RuntimeError, match="background must be"):
        svox.composite(x, g, torch.rand(3, 6))


def test_abi_refusals():
    import ctypes as C

    class Scan(C.Structure):
        _fields_ = [("values", C.c_void_p), ("thickness", C.c_void_p), ("initial", C.c_void_p),
                    ("offsets", C.c_void_p), ("B", C.c_int64), ("T", C.c_int64),
                    ("values_row", C.c_int64), ("values_step", C.c_int64),
                    ("thickness_row", C.c_int64), ("thickness_step", C.c_int64),
                    ("initial_row", C.c_int64), ("C", C.c_int32), ("H", C.c_int32),
                    ("values_type", C.c_int32), ("thickness_type", C.c_int32),
                    ("reverse", C.c_int32), ("weighted", C.c_int32),
                    ("last_only", C.c_int32), ("layout", C.c_int32)]

    lib = csrc.library()
    lib.svoxb_gated_scan_kept.restype = lib.svoxb_gated_scan_workspace.restype = C.c_int64

    def call(**k):
        s = Scan(16, 16, None, None, 2, 3, 12, 4, 3, 1, 0, 4, 1, 0, 0, 0, 0, 1, 0)
        for name, v in k.items():
            setattr(s, name, v)
        return lib.svoxb_gated_scan(C.byref(s), None, None, None, None, None), s

    assert call()[0] == 1                                   # no `last`
    assert call(values=None)[0] == 1 and call(thickness=None)[0] == 1
    assert call(B=-1)[0] == 2 and call(T=-1)[0] == 2 and call(C=0)[0] == 2 and call(H=3)[0] == 2
    assert call(values_type=3)[0] == 3 and call(thickness_type=1)[0] == 3
    assert call(T=1 << 41)[0] == 8
    assert call(last_only=0)[0] == 1                        # no states
    assert call(layout=3)[0] == 4
    assert call(B=0)[0] == 0                                # nothing to do
    assert lib.svoxb_gated_scan(None, None, None, None, None, None) == 1
    s = call(H=3)[1]
    assert lib.svoxb_gated_scan_kept(C.byref(s)) == -1
    assert lib.svoxb_gated_scan_workspace(C.byref(s), 1) == -1
    assert lib.svoxb_gated_scan_backward(C.byref(s), None, None, None, None, None, None, None,
                                         None) == 2
    s = call()[1]
    assert lib.svoxb_gated_scan_backward(C.byref(s), None, None, None, None, None, None, None,
                                         None) == 1         # no kept states


def scan_struct():
    import ctypes as C

    class Scan(C.Structure):
        _fields_ = [("values", C.c_void_p), ("thickness", C.c_void_p), ("initial", C.c_void_p),
                    ("offsets", C.c_void_p), ("B", C.c_int64), ("T", C.c_int64),
                    ("values_row", C.c_int64), ("values_step", C.c_int64),
                    ("thickness_row", C.c_int64), ("thickness_step", C.c_int64),
                    ("initial_row", C.c_int64), ("C", C.c_int32), ("H", C.c_int32),
                    ("values_type", C.c_int32), ("thickness_type", C.c_int32),
                    ("reverse", C.c_int32), ("weighted", C.c_int32),
                    ("last_only", C.c_int32), ("layout", C.c_int32)]

    return Scan


@pytest.mark.parametrize("C", [3, 32, 35, 120, 128, 136, 200, 256, 264])
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_what_is_kept_follows_the_layout(C, kind):
    """What the forward pass keeps goes by sizes, types and `layout`, not by where the arrays lie."""
    import ctypes as ct
    lib = csrc.library()
    lib.svoxb_gated_scan_kept.restype = ct.c_int64
    B, T, size = 1000, 64, 4 if kind == 0 else 2
    wide = (C + 5) // 2 * 2 + 1
    for offsets in (None, 16):
        kept = {}
        for address, step in ((1 << 20, C), ((1 << 20) + size, C), (1 << 20, wide)):
            s = scan_struct()(address, 1 << 20, None, offsets, B, T * B if offsets else T, T * step,
                              step, T, 1, 0, C, 1, kind, 0, 1, 0, 1, 0)
            layout = lib.svoxb_gated_scan_layout(ct.byref(s))
            mine = lib.svoxb_gated_scan_kept(ct.byref(s))
            s.layout = layout
            assert lib.svoxb_gated_scan_layout(ct.byref(s)) == layout
            assert lib.svoxb_gated_scan_kept(ct.byref(s)) == mine
            assert kept.setdefault(layout, mine) == mine, (layout, kept, mine)


def off_boundary(t):
    """The same values, one element off a 16-byte boundary."""
    to = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    to[1:] = t.detach().flatten()
    return to[1:].view(t.shape)


def on_columns(t):
    """The same values in rows of a wider array."""
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    wide[..., 1:-2] = t.detach()
    return wide[..., 1:-2]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("C", [120, 136, 200, 256, 264])
@pytest.mark.parametrize("many", [False, True])
def test_features_saved_elsewhere(cuda_device, C, dtype, many):
    """Wide features in 16 bits whose saved tensors lie elsewhere than the forward's, either way: on
    their boundaries, off them, in a wider array, by way of the host."""
    gen = torch.Generator().manual_seed(C)
    n = torch.tensor([30, 0, 77, 5, 1, 200] + [0, 1, 0] * (200 if many else 0))
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(cuda_device)
    x, g = inputs(gen, (int(n.sum()),), C, 1, dtype, F32, cuda_device)
    d = torch.randn(n.numel(), C, generator=gen).to(cuda_device)
    want = reference(x, g, None, offsets, True, False, None, d)
    places = [lambda t: t.detach().clone(), off_boundary, on_columns]
    for place in places:
        def moved(to):
            return lambda t: to(t) if t.dtype == dtype else t
        hooks = [torch.autograd.graph.saved_tensors_hooks(lambda t: t, moved(to)) for to in places]
        for hook in [*hooks, torch.autograd.graph.save_on_cpu()]:
            leaves = [place(x).requires_grad_(True), g.detach().clone().requires_grad_(True)]
            with hook:
                out = svox.composite(*leaves, offsets=offsets)
            close("last", out, want["last"])
            for name, got in zip(("d_values", "d_thickness"), torch.autograd.grad(out, leaves, d)):
                close(name, got, want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("C,H", [(3, 1), (32, 1), (200, 1), (64, 8), (5, 5)])
def test_saved_tensors_in_another_order(cuda_device, C, H):
    """A hook hands back the saved tensors with strides of its own, or something else altogether."""
    gen = torch.Generator().manual_seed(C)
    n = torch.tensor([30, 0, 77, 5, 1])
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(cuda_device)
    x, g = inputs(gen, (int(n.sum()),), C, H, F32, F32, cuda_device)
    h0 = torch.randn(5, C, generator=gen).to(cuda_device)
    d = torch.randn(5, C, generator=gen).to(cuda_device)
    want = reference(x, g, h0, offsets, True, False, None, d)

    def strided(t):
        out = torch.empty(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=t.device)
        out[..., ::2] = t
        return out[..., ::2]

    def transposed(t):
        return t.transpose(0, -1).clone(memory_format=torch.contiguous_format).transpose(0, -1)

    def grads(unpack):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, g, h0)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            if H == 1:
                out = svox.composite(*leaves, offsets)
            else:
                out = svox.gated_scan(*leaves, offsets, reverse=True)[1]
        return torch.autograd.grad(out, leaves, d)

    for to in (strided, transposed):
        for name, got in zip(("d_values", "d_thickness", "d_initial"), grads(to)):
            close(name, got, want[name])
    for to in (lambda t: t.double() if t.dtype == F32 else t, lambda t: t[:-1], lambda t: t.cpu(),
               lambda t: t[None]):
        with pytest.raises(RuntimeError, match="saved tensor"):
            grads(to)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [1, 3, 4, 32, 300])
@pytest.mark.parametrize("place", [0, 1, 2])
def test_an_opaque_sample_of_infinite_value(cuda_device, C, place):
    """Its thickness has no gradient (nothing is behind it, and none of it gets past): wherever the
    arrays lie."""
    gen = torch.Generator().manual_seed(C)
    x, g = inputs(gen, (9, 40), C, 1, F32, F32, cuda_device)
    at = [0, 1, 2, 3, 13, 17, 22, 31, 39]
    for row, k in enumerate(at):
        g[row, k] = float("inf")
        x[row, k, C // 2] = float("inf")
    bg = torch.rand(9, C, generator=gen).to(cuda_device)
    d = torch.rand(9, C, generator=gen).to(cuda_device) + 0.5
    where = (lambda t: t.detach().clone(), off_boundary, on_columns)[place]
    leaves = [where(t).requires_grad_(True) for t in (x, g, bg)]
    out = svox.composite(*leaves)
    dx, dg, db = torch.autograd.grad(out, leaves, d)
    want = reference(x, g, bg, None, True, False, None, d)
    for row, k in enumerate(at):
        assert out[row, C // 2] == float("inf")
        assert (dg[row, k:] == 0).all() and (dx[row, k + 1:] == 0).all() and (db[row] == 0).all()
        part = slice(row, row + 1)
        close("d_values", dx[part], [v[part] for v in want["d_values"]])


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,C,H", [(1, 6000, 64, 64), (1, 6000, 64, 2), (2, 700, 70, 70), (3, 90, 6, 1),
                                     (3, 90, 6, 3), (1, 6000, 5, 1), (400, 40, 8, 8), (40, 300, 130, 1)])
@pytest.mark.parametrize("thick", [0.4, 20.0])
def test_not_a_number_stays(cuda_device, B, T, C, H, thick):
    """Only a step that is opaque by itself ends it, not many that together leave nothing of a finite
    amount, however the steps are shared out: forwards for the states, backwards for the gradients."""
    gen = torch.Generator().manual_seed(T + C)
    for bad in (float("nan"), float("inf")):
        x, g = inputs(gen, (B, T), C, H, F32, F32, cuda_device)
        g = torch.rand(g.shape, generator=gen).to(cuda_device) * thick + thick / 2
        x[:, 0] = bad
        h0 = torch.rand(B, C, generator=gen).to(cuda_device)
        d_states = torch.rand(B, T, C, generator=gen).to(cuda_device)
        leaves = [t.clone().requires_grad_(True) for t in (x, g, h0)]
        states, last = svox.gated_scan(*leaves)
        assert not states.isfinite().any() and not last.isfinite().any()
        if bad == float("inf"):
            assert (last == bad).all() and (states == bad).all()
        x[:, 0] = 1.0
        leaves = [t.clone().requires_grad_(True) for t in (x, g, h0)]
        states, last = svox.gated_scan(*leaves)
        d_states[:, -1] = bad
        grads = torch.autograd.grad((states, last), leaves, (d_states, torch.rand_like(last)))
        for t in grads[:1] + grads[2:]:
            assert not t.isfinite().any()
            if bad == float("inf"):
                assert (t == bad).all()
        # an opaque step ends it
        k = T * 2 // 3
        g[:, k] = float("inf")
        x[:, 0] = bad
        states, last = svox.gated_scan(x, g, h0)
        assert not states[:, :k].isfinite().any()
        assert states[:, k:].isfinite().all() and last.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("C", [1, 3, 32, 64, 300])
@pytest.mark.parametrize("premultiplied", [False, True])
def test_not_a_number_in_front_of_an_opaque_sample(cuda_device, C, premultiplied):
    """The colour is not a number then, but what the opaque sample hides has no part in it: no
    gradient, in `composite` as in `gated_scan`, whatever the sums of thickness in between."""
    gen = torch.Generator().manual_seed(C)
    x, g = inputs(gen, (8, 300), C, 1, F32, F32, cuda_device)
    g = g.clamp(min=0.01)
    at = [(0, 1), (0, 2), (5, 7), (3, 130), (17, 40), (60, 299), (128, 129), (100, 255)]
    for row, (k, opaque) in enumerate(at):
        g[row, k] = float("nan")
        g[row, opaque] = float("inf")
    g[3, 40:130] = 30.0                 # (together far more than leaves nothing of a finite amount)
    bg = torch.rand(8, C, generator=gen).to(cuda_device)
    d = torch.randn(8, C, generator=gen).to(cuda_device)
    for place in (lambda t: t.detach().clone(), off_boundary, on_columns):
        leaves = [place(t).requires_grad_(True) for t in (x, g, bg)]
        for call in (lambda *v: svox.composite(*v, premultiplied=premultiplied),
                     lambda *v: svox.gated_scan(*v, reverse=True, premultiplied=premultiplied)[1]):
            out = call(*leaves)
            dx, dg, db = torch.autograd.grad(out, leaves, d)
            for row, (k, opaque) in enumerate(at):
                assert (dx[row, opaque + 1:] == 0).all() and (dg[row, opaque + 1:] == 0).all()
                assert (db[row] == 0).all() and dx[row, :k].isfinite().all()
                # what is in front of it is not hidden, where anything of the light gets there (a
                # composite counts nothing where 32 bits hold nothing of it)
                if torch.exp(-g[row, :k].double().sum()) > 2.0 ** -126:
                    assert out[row].isnan().all() and dx[row, k + 1:opaque + 1].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("C,H", [(3, 1), (32, 1), (300, 1), (64, 4), (70, 70)])
@pytest.mark.parametrize("premultiplied", [False, True])
def test_hidden_samples_have_no_gradient(cuda_device, C, H, premultiplied):
    """Behind an opaque sample neither a value nor a thickness has one, whatever the values are."""
    gen = torch.Generator().manual_seed(C)
    x, g = inputs(gen, (4, 120), C, H, F32, F32, cuda_device)
    at = [0, 9, 50, 118]
    for row, k in enumerate(at):
        g[row, k] = float("inf")
        x[row, k + 1::2] = float("nan")
        x[row, k + 3::4] = float("inf")
    bg = torch.full((4, C), float("nan"), device=cuda_device)
    d = torch.randn(4, C, generator=gen).to(cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, g, bg)]
    out = svox.composite(*leaves, premultiplied=premultiplied)
    dx, dg, db = torch.autograd.grad(out, leaves, d)
    assert (db == 0).all()
    for row, k in enumerate(at):
        assert (dx[row, k + 1:] == 0).all() and (dg[row, k + 1:] == 0).all()
        part = slice(row, row + 1), slice(0, k + 1)
        want = reference(x[part], g[part], None, None, True, premultiplied, None, d[part[0]])
        close("d_values", dx[part], want["d_values"])
        close("d_thickness", dg[part], want["d_thickness"])


@pytest.mark.gpu
@pytest.mark.parametrize("C,H", [(64, 64), (64, 8), (3, 1)])
@pytest.mark.parametrize("premultiplied", [False, True])
def test_thin_gates_over_a_long_sequence(cuda_device, C, H, premultiplied):
    """2^17 steps of a thickness around 1e-5: errors of single steps that lie to one side would add up
    to T of them.  Rounded to nearest, a = exp(-g) and the sum of a step are off by at most u / 2 each
    of a state that stays within 1 (weighted beforehand: of the sum of its terms), to either side
    as g varies: a random walk of 2 T such steps, each of variance u^2 / 12, that leaves
    6 sqrt(T / 6) u with a probability of 2e-9; the weights' own error, 3 u of each, adds 3 u.  A product
    of numbers 1 - p, 1 - q just below 1 rounds up or down to 1 - p - q wherever p q is below u / 2: each
    stretch of 8 steps loses its 28 pairs, 28 g^2, and the first few of the folds of a range of steps
    half a u each, of up to 256 ranges below 1.5 g^2 for every step of all: 5 T g^2 together."""
    gen = torch.Generator().manual_seed(C + H)
    T = 1 << 17
    g = (torch.rand(1, T, H, generator=gen) * 1.9 + 0.1) * 1e-5
    x = torch.full((1, T, C), 0.75)
    if premultiplied:
        x *= 1e-5
    h0 = torch.full((1, C), 0.5)
    args = [t.to(cuda_device).requires_grad_(True) for t in (x, g, h0)]
    states, last = svox.gated_scan(*args, premultiplied=premultiplied)
    d = torch.ones(1, C, device=cuda_device)
    grads = torch.autograd.grad(last, args, d)
    gates = g[0].double().repeat_interleave(C // H, 1)
    upto = gates.cumsum(0)
    if premultiplied:       # (a sum of positive terms by the share that remains of each)
        want = torch.exp(-upto[-1]) * 0.5 + \
            (torch.exp(upto - upto[-1]) * x[0].double()).sum(0)
        mid = torch.exp(-upto[T // 2]) * 0.5 + \
            (torch.exp(upto[:T // 2 + 1] - upto[T // 2]) * x[0, :T // 2 + 1].double()).sum(0)
    else:                   # (a constant value: what is not the first state is that)
        want, mid = (0.75 - 0.25 * torch.exp(-upto[k]) for k in (-1, T // 2))
    tol = ((6 * (T / 6) ** 0.5 + 3) * U + 5 * T * 1.05e-5 ** 2) * max(1.0, float(want.max()))
    assert (last[0].cpu().double() - want).abs().max() <= tol
    assert (states[0, T // 2].cpu().double() - mid).abs().max() <= tol
    assert (grads[2][0].cpu().double() - torch.exp(-upto[-1])).abs().max() <= tol
    through = torch.exp(upto - upto[-1])
    dx = through if premultiplied else through * -torch.expm1(-gates)
    assert ((grads[0][0].cpu().double() - dx).abs() <= tol * dx / through).all()


def test_sizes_beyond_the_maximum_are_refused():
    """More channels than the kernels count, beyond 32 bits too."""
    for C in ((1 << 24) + 1, 1 << 31, (1 << 32) + 64):
        x = torch.zeros(1).expand(1, 1, C)
        with pytest.raises(RuntimeError, match="channels"):
            svox.gated_scan(x, torch.zeros(1, 1))
        with pytest.raises(RuntimeError, match="channels"):
            svox.composite(x, torch.zeros(1, 1, 1).expand(1, 1, C))


@pytest.mark.gpu
@pytest.mark.parametrize("C,H", [(3, 1), (64, 64)])
def test_views_of_negatives(cuda_device, C, H):
    """Imaginary parts of a conjugate, whose memory holds their negatives: inputs and gradients."""
    gen = torch.Generator().manual_seed(C)
    x, g = inputs(gen, (2, 40), C, H, F32, F32, cuda_device)
    h0 = torch.randn(2, C, generator=gen).to(cuda_device)
    d = torch.randn(2, C, generator=gen).to(cuda_device)

    def view(t):
        t = torch.complex(t, -t).conj().imag
        assert t.is_neg()
        return t

    for to in (view, lambda t: torch._neg_view(-t)):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, g, h0)]
        plain = svox.gated_scan(*leaves)
        want = torch.autograd.grad(plain[1], leaves, d)
        states, last = svox.gated_scan(*[to(t.detach()) for t in leaves])
        assert torch.equal(states, plain[0]) and torch.equal(last, plain[1])
        for a, b in zip(torch.autograd.grad(svox.gated_scan(*leaves)[1], leaves, to(d)), want):
            assert torch.equal(a, b)
        with torch.autograd.graph.saved_tensors_hooks(
                lambda t: t, lambda t: to(t) if t.dtype == F32 else t):
            last = svox.gated_scan(*leaves)[1]
        for a, b in zip(torch.autograd.grad(last, leaves, d), want):
            assert torch.equal(a, b)
