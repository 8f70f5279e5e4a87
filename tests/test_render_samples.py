"""The operators together: records looked up at samples along rays (in the tree or in a quantised
cache), weighted and composited, against the same in 64 bits, and against the march."""
import pytest
import torch

import svox_b200 as svox
from svox_b200 import csrc, workloads
from svox_b200.sh import eval_sh_bases

U = 2.0 ** -24


def scene(fmt, dev, data_dim=None):
    gen = torch.Generator().manual_seed(11)
    tree = svox.N3Tree(data_format=fmt, data_dim=data_dim, init_refine=3, device=dev)
    d = torch.randn(tree.data.shape, generator=gen)
    d[..., -1] = torch.rand(d.shape[:-1], generator=gen) * 12 - 2       # some negative
    tree.data.data.copy_(d)
    rays = workloads.sphere_rays(70, gen, 1.5, 0.3, 0.7)
    return tree, svox.Rays(*[t.to(dev) for t in rays]), gen


def plain(tree, data, rays, ids, ray, rows, lengths, renderer):
    """In 64 bits: colours, and the sum of magnitudes that their rounding goes by."""
    K = tree.data_dim
    rec = data.double().reshape(-1, K)[ids]
    sigma = rec[:, -1]
    sigma = torch.nn.functional.softplus(sigma - 1) if renderer.density_softplus else sigma.relu()
    rgb = rec[:, :-1]
    n = tree.data_format.basis_dim
    if n > 0:
        basis = eval_sh_bases(int(round(n ** 0.5)) - 1, rays.viewdirs.double())
        hi = renderer.max_comp if renderer.max_comp >= 0 else n + renderer.max_comp
        some = slice(renderer.min_comp, hi + 1)
        rgb = (rgb.reshape(-1, 3, n)[..., some] * basis[ray][:, None, some]).sum(-1)
    pad = renderer.rgb_padding
    rgb = torch.sigmoid(rgb) * (1 + 2 * pad) - pad
    g = sigma * lengths.double()
    out = []
    for lo, hi in rows:
        t = torch.cat([g.new_zeros(1), g[lo:hi].cumsum(0)])
        w = torch.exp(-t[:-1]) * -torch.expm1(-g[lo:hi])
        out.append((w[:, None] * rgb[lo:hi]).sum(0) +
                   torch.exp(-t[-1]) * renderer.background_brightness)
    return torch.stack(out)


def tolerance(T):
    """Colours lie within 1 and weights sum to 1.  A sample's colour is off by 60 u (a sum of up to
    16 products, each of magnitude below 8, through a sigmoid of slope below 1 / 4, 16 * 8 / 4 u, and
    the sigmoid itself, below 28 u); its weight by 20 u and by the roundings of the thickness in
    front of it, T u g exp(-g) a step (below 1 together for every 2.7 of them)."""
    return (60 + 20 + T) * U


CASES = [("SH4", None, {}), ("SH9", None, {"min_comp": 1, "max_comp": 6}),
         ("SH16", None, {"rgb_padding": 0.01, "background_brightness": 0.25}),
         ("SH1", None, {"density_softplus": True}), ("RGBA", 4, {}), ("RGBA", 7, {})]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,dim,more", CASES, ids=str)
@pytest.mark.parametrize("packed", [False, True])
def test_render_samples(cuda_device, fmt, dim, more, packed):
    tree, rays, gen = scene(fmt, cuda_device, dim)
    renderer = svox.VolumeRenderer(tree, **more)
    B, T = 70, 90
    if packed:
        n = torch.randint(0, T, (B,), generator=gen)
        n[3] = n[17] = 0
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)])
        rows = list(zip(offsets[:-1].tolist(), offsets[1:].tolist()))
        depths = torch.cat([torch.linspace(0.6, 2.4, int(k)) for k in n])
        ray = torch.repeat_interleave(torch.arange(B), n)
        offsets = offsets.to(cuda_device)
    else:
        depths = torch.linspace(0.6, 2.4, T).repeat(B, 1)
        ray = torch.arange(B).repeat_interleave(T)
        rows, offsets = [(b * T, b * T + T) for b in range(B)], None
    lengths = torch.rand(depths.shape, generator=gen) * 0.05
    depths, lengths = depths.to(cuda_device), lengths.to(cuda_device).requires_grad_(True)
    out = renderer.render_samples(rays, depths, lengths, offsets)
    ray = ray.to(cuda_device)
    points = torch.addcmul(rays.origins[ray], depths.reshape(-1, 1), rays.dirs[ray])
    ids = tree(points, want_node_ids=True)[1]
    data = tree.data.detach().double().requires_grad_(True)
    len64 = lengths.detach().double().reshape(-1).requires_grad_(True)
    want = plain(tree, data, rays, ids, ray, rows, len64, renderer)
    assert out.shape == want.shape
    assert (out.double() - want).abs().max() <= tolerance(T)
    d = torch.randn(want.shape, generator=gen).to(cuda_device)
    got = torch.autograd.grad(out, [tree.data, lengths], d)
    ref = torch.autograd.grad(want, [data, len64], d.double())
    # a record's gradient sums over up to N samples whose terms are off by as much as a colour, times
    # what they are multiplied with: d (below 5), basis (below 2), density (10) or length
    for g, r, scale in ((got[0], ref[0], 10), (got[1].reshape(-1), ref[1], 50 * 3)):
        assert (g.double() - r).abs().max() <= tolerance(T) * scale * max(1.0, r.abs().max().item())
    # the quantised cache: as a tree that holds its values
    if fmt.startswith("SH") or dim == 4:
        for dtype in (torch.int8, torch.float8_e4m3fn):
            cache = svox.RecordCache(tree, dtype=dtype)
            with torch.no_grad():
                a = renderer.render_samples(rays, depths, lengths, offsets, cache=cache)
                kept = tree.data.data.clone()
                tree.data.data.copy_(cache.read().reshape(kept.shape))
                b = renderer.render_samples(rays, depths, lengths, offsets)
                tree.data.data.copy_(kept)
            assert torch.equal(a, b)
    assert csrc.device_status() == 0


@pytest.mark.gpu
def test_samples_where_the_march_takes_them(cuda_device):
    """One sample for each leaf that a ray crosses is the march itself (but for the step that it
    adds to every leaf)."""
    tree, _, gen = scene("SH4", cuda_device)
    renderer = svox.VolumeRenderer(tree, step_size=1e-5)
    B, n = 16, 16
    dirs = torch.tensor([[1.0, 0.0, 0.0]]).repeat(B, 1).to(cuda_device)
    origins = torch.rand(B, 3, generator=gen).to(cuda_device)
    origins[:, 0] = -0.5
    rays = svox.Rays(origins, dirs, dirs)
    depths = (0.5 + (torch.arange(n) + 0.5) / n).repeat(B, 1).to(cuda_device)
    lengths = torch.full_like(depths, 1.0 / n)
    with torch.no_grad():
        a, b = renderer.render_samples(rays, depths, lengths), renderer(rays)
    # each leaf's thickness is off by at most 12 * 1e-5, a colour by at most the sum of those
    assert (a - b).abs().max() <= n * 12 * 1e-5 + tolerance(n)


@pytest.mark.gpu
def test_training_through_samples(cuda_device):
    """A few steps of gradient descent run, eagerly and as a captured graph, with the same result."""
    tree, rays, gen = scene("SH4", cuda_device)
    renderer = svox.VolumeRenderer(tree)
    depths = torch.linspace(0.6, 2.4, 40).repeat(70, 1).to(cuda_device)
    lengths = torch.full_like(depths, 0.045)
    target = torch.rand(70, 3, generator=gen).to(cuda_device)

    def grad():
        out = renderer.render_samples(rays, depths, lengths)
        return torch.autograd.grad(((out - target) ** 2).sum(), [tree.data])[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            grad()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = grad()
    for _ in range(3):
        graph.replay()
        want = grad()
        assert want.isfinite().all()
        # (the query's backward sums a leaf's rows in no fixed order: at most 2800 terms)
        assert (held - want).abs().max() <= 2800 * U * want.abs().max()
        with torch.no_grad():
            tree.data -= 0.1 * want


def test_refusals():
    tree = svox.N3Tree(data_format="SH4")
    renderer = svox.VolumeRenderer(tree)
    z = torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="no CPU render path"):
        renderer.render_samples(svox.Rays(z, z, z), torch.zeros(2, 4), torch.zeros(2, 4))


@pytest.mark.gpu
def test_refusals_gpu(cuda_device):
    tree, rays, _ = scene("SH4", cuda_device)
    renderer = svox.VolumeRenderer(tree)
    d = torch.zeros(70, 4, device=cuda_device)
    o = torch.zeros(71, dtype=torch.int64, device=cuda_device)
    for args in ((rays, d[:5], d[:5]), (rays, d, d[:, :3]), (rays, d[0], d[0]),
                 (rays, d, d, o), (rays, d[0], d[0], o[:5])):
        with pytest.raises(RuntimeError, match="depths and lengths"):
            renderer.render_samples(*args)
    lobes = svox.N3Tree(data_format="SG2", extra_data=torch.ones(2, 4), device=cuda_device)
    with pytest.raises(RuntimeError, match="RGBA and SH"):
        svox.VolumeRenderer(lobes).render_samples(rays, d, d)
    none = svox.Rays(*[t[:0] for t in rays])
    assert renderer.render_samples(none, d[:0], d[:0]).shape == (0, 3)
    assert renderer.render_samples(none, d[0, :0], d[0, :0], o[:1]).shape == (0, 3)
    assert (renderer.render_samples(rays, d[:, :0], d[:, :0]) == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_buffers_that_are_not_full(cuda_device, junk):
    """Room for more samples than there are, and whatever lies there: the same colours and gradients as
    where only the samples themselves are given, and no gradient in the room that is left."""
    tree, rays, gen = scene("SH4", cuda_device)
    renderer = svox.VolumeRenderer(tree)
    n = torch.randint(0, 60, (70,), generator=gen)
    n[0] = n[69] = 0            # (the rays next to the room, and nothing of them is known)
    for t in rays:
        t[0] = t[69] = float("nan")
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)])
    N, lo, hi = int(offsets[-1]), 13, 29
    some = torch.cat([torch.linspace(1.2, 1.8, int(k)) for k in n]), torch.rand(N, generator=gen) * 0.05
    d = torch.randn(70, 3, generator=gen).to(cuda_device)
    got = []
    for room in (False, True):
        depths, lengths, o = *some, offsets
        if room:
            def wide(t):
                out = torch.full((lo + N + hi,), junk)
                out[lo:lo + N] = t
                return out
            depths, lengths, o = wide(depths), wide(lengths), offsets + lo
        lengths = lengths.to(cuda_device).requires_grad_(True)
        out = renderer.render_samples(rays, depths.to(cuda_device), lengths, o.to(cuda_device))
        got.append([out, *torch.autograd.grad(out, [tree.data, lengths], d)])
    assert all(t.isfinite().all() for t in got[1])
    # (samples at another place of the arrays are summed in another order: either side is off from the
    # sums by at most the tolerances of test_render_samples, with its scales, so twice those between them)
    for a, b, scale in ((got[0][0], got[1][0], 1), (got[0][1], got[1][1], 10),
                        (got[0][2], got[1][2][lo:lo + N], 50 * 3)):
        assert (a - b).abs().max() <= 2 * tolerance(60) * scale * max(1.0, a.abs().max().item())
    assert (got[1][2][:lo] == 0).all() and (got[1][2][lo + N:] == 0).all()
    assert csrc.device_status() == 0
