"""Quantised leaf records against a plain quantiser in 64 bits.

The scales are powers of two, so scaling is exact and a code is the nearest of its type: the kernels
have to agree to the bit, and no tolerance is needed."""
import math

import numpy as np
import pytest
import torch

import svox_b200 as svox
from svox_b200 import csrc

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def nearest(y, dtype):
    """Nearest code (ties to even) of magnitudes within range, as values."""
    if dtype == INT8:
        return torch.round(y)
    # e4m3: steps of an eighth of the power of two below, of 2^-9 under 2^-6
    size = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0)
    step = torch.exp2(size - 3)
    return torch.round(y / step) * step


def held(rows, group, dtype):
    """What records of these rows read as, in 64 bits (rows of one group at a time)."""
    rows = rows.detach().cpu().double()
    out = rows.clone()
    out[:, -1] = rows[:, -1].float().half().double()
    top = 127.0 if dtype == INT8 else 448.0
    K = rows.shape[1]
    for c in range(0, K - 1, group):
        part = rows[:, c:min(c + group, K - 1)]
        for q, row in enumerate(part):
            most = row.abs().max().item()
            if not math.isfinite(most):
                out[q, c:c + part.shape[1]] = float("nan")
                continue
            e = -126
            if most > 0:
                e = max(e, math.frexp(most)[1] - 20)
                while nearest(torch.tensor(most * 2.0 ** -e, dtype=torch.float64), INT8).item() \
                        > top if dtype == INT8 else most * 2.0 ** -e > top:
                    e += 1
            out[q, c:c + part.shape[1]] = nearest(row * 2.0 ** -e, dtype) * 2.0 ** e
    return out


def same(got, want, dtype=None):
    """Equal to the bit, NaN where it is (to 16 bits: the value rounded once)."""
    got = got.detach().cpu()
    want = want.float().to(got.dtype)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want[~nan])


def make_tree(fmt, dev, data_dim=None, refine=2, N=2, seed=0, **more):
    gen = torch.Generator().manual_seed(seed)
    tree = svox.N3Tree(N=N, data_dim=data_dim, data_format=fmt, init_refine=refine, device=dev,
                       **more)
    if N == 2 and refine >= 1:
        tree[torch.rand(20, 3, generator=gen).to(dev)].refine()
    d = tree.data.data
    rows = torch.randn(d.shape, generator=gen) * torch.exp2(
        torch.randint(-12, 12, d.shape[:-1], generator=gen))[..., None]
    rows[..., -1] = torch.rand(d.shape[:-1], generator=gen) * 60
    d.copy_(rows)
    return tree


def flat(tree):
    return tree.data.detach().reshape(-1, tree.data_dim)


FORMATS = [("SH1", None), ("SH4", None), ("SH9", None), ("SH16", None), ("SH25", None),
           ("RGBA", 4), ("RGBA", 2), ("RGBA", 34), ("RGBA", 129), ("RGBA", 1024), ("SG7", None)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,dim", FORMATS, ids=str)
@pytest.mark.parametrize("dtype", [INT8, E4M3], ids=str)
def test_whole_tree(cuda_device, fmt, dim, dtype):
    extra = torch.ones(7, 4) if fmt == "SG7" else None
    tree = make_tree(fmt, cuda_device, dim, refine=1, extra_data=extra)
    cache = svox.RecordCache(tree, dtype=dtype)
    want = held(flat(tree), cache.group, dtype)
    same(cache.read(), want)
    gen = torch.Generator().manual_seed(1)
    points = torch.rand(700, 3, generator=gen).to(cuda_device)
    ids = tree(points, want_node_ids=True)[1]
    for t in (F32, BF16, F16):
        same(cache(points, dtype=t), want[ids.cpu()])
        same(cache.read(ids, dtype=t), want[ids.cpu()])
    bound = cache.records.shape[1]
    assert bound == csrc.record_bytes(tree.data_dim, cache.group)
    assert csrc.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 2, 5, 27, 100])
@pytest.mark.parametrize("dtype", [INT8, E4M3], ids=str)
def test_groups(cuda_device, group, dtype):
    tree = make_tree("SH9", cuda_device, refine=1)
    cache = svox.RecordCache(tree, dtype=dtype, group=group)
    same(cache.read(), held(flat(tree), group, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [INT8, E4M3], ids=str)
def test_borders_of_the_scale(cuda_device, dtype):
    """Largest magnitudes on and beside the border where the scale changes, ties, zeros of both
    signs, the smallest and largest floats, and values that are not finite."""
    base = [0.0, -0.0, 1.0, 127.0, 127.49999, 127.5, 127.50001, 128.0, 448.0, 448.00003, 464.0, 480.0,
            255.0, 1e-38, 1e-45, 3e38, 6e-8, 0.3]
    rows = []
    for most in base:
        for scale in (1.0, 2.0 ** -40, 2.0 ** 60):
            v = np.float32(most * scale) if most * scale < 3.4e38 else np.float32(3.4e38)
            rows.append([v, -v / 3, v * 0.5, v / 254, -v * 0.0039, 0.0, -0.0, v * 0.99, v / 7, 5.0])
    inf, nan = float("inf"), float("nan")
    rows += [[inf] + [1.0] * 8 + [2.0], [1.0] * 8 + [nan, inf], [nan] * 9 + [nan],
             [1.0] * 9 + [70000.0], [-inf, nan] + [0.0] * 7 + [-1e-9], [1.0] * 9 + [65519.9]]
    values = torch.tensor(np.array(rows, np.float32), device=cuda_device)
    tree = make_tree("RGBA", cuda_device, 10, refine=1)
    cache = svox.RecordCache(tree, dtype=dtype)
    ids = torch.randperm(len(cache))[:values.shape[0]].to(cuda_device)
    cache.write(ids, values)
    same(cache.read(ids), held(values, 9, dtype))
    # in groups of 4 and 5: what is not finite spoils its own group
    cache = svox.RecordCache(tree, dtype=dtype, group=4)
    cache.write(ids, values)
    same(cache.read(ids), held(values, 4, dtype))


@pytest.mark.gpu
def test_error_is_half_a_step(cuda_device):
    tree = make_tree("SH16", cuda_device, refine=2)
    rows = flat(tree).cpu()
    colour = rows[:, :-1].reshape(-1, 3, 16).double()
    most = colour.abs().amax(-1, keepdim=True)
    got = svox.RecordCache(tree).read().cpu().double()[:, :-1].reshape(colour.shape)
    # half of a step of at most most / 63.75 (the largest code is above 63)
    assert ((got - colour).abs() <= most / 127.5).all()
    got = svox.RecordCache(tree, dtype=E4M3).read().cpu().double()[:, :-1].reshape(colour.shape)
    # e4m3 has half a step of 2^-4 of the value, or 2^-10 of a scale below most / 224
    assert ((got - colour).abs() <= (colour.abs() * 2.0 ** -4).maximum(most / 224 * 2.0 ** -10)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["SH4", "SH9", "SH25"])
@pytest.mark.parametrize("values", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("by", ["points", "ids"])
def test_writes(cuda_device, fmt, values, by):
    """Rows in any order, several for a leaf (the last counts), everything else as it was."""
    tree = make_tree(fmt, cuda_device, refine=2)
    gen = torch.Generator().manual_seed(2)
    for dtype, Q in ((INT8, 1), (E4M3, 33), (INT8, 1501), (E4M3, 40000)):
        cache = svox.RecordCache(tree, dtype=dtype)
        before = cache.records.clone()
        points = torch.rand(Q, 3, generator=gen).to(cuda_device)
        if Q > 1000:
            points[::7] = points[3]         # one leaf, many times
        ids = tree(points, want_node_ids=True)[1]
        new = torch.randn(Q, tree.data_dim, generator=gen).to(cuda_device, values)
        if by == "points":
            cache.set(points, new)
        else:
            cache.write(ids, new)
        last = {}
        for q, i in enumerate(ids.tolist()):
            last[i] = q
        where = torch.tensor(list(last), device=cuda_device)
        rows = new[torch.tensor(list(last.values()), device=cuda_device)]
        pick = slice(0, 2000)
        same(cache.read(where[pick]), held(rows[pick], cache.group, dtype))
        rest = torch.ones(len(cache), dtype=torch.bool, device=cuda_device)
        rest[where] = False
        assert torch.equal(cache.records[rest], before[rest])
        assert (cache._owner == 0).all()
        # the same rows again, the other way round: now the first ones count
        if Q > 1000:
            cache.write(ids.flip(0), new.flip(0))
            first = {}
            for q, i in reversed(list(enumerate(ids.tolist()))):
                first[i] = q
            rows = new[torch.tensor([first[i] for i in last], device=cuda_device)]
            same(cache.read(where[pick]), held(rows[pick], cache.group, dtype))


@pytest.mark.gpu
def test_other_trees_and_frames(cuda_device):
    """N = 3, a tree off the unit cube, local coordinates, points outside, a jump table."""
    gen = torch.Generator().manual_seed(3)
    for tree in (make_tree("SH4", cuda_device, N=3, refine=1),
                 make_tree("SH4", cuda_device, refine=4, radius=[1.0, 2.0, 3.0],
                           center=[0.5, -1.0, 4.0])):
        cache = svox.RecordCache(tree)
        for Q in (500, 1 << 18):
            points = (torch.rand(Q, 3, generator=gen) * 8 - 3).to(cuda_device)
            ids = tree(points, want_node_ids=True)[1]
            assert torch.equal(cache(points), cache.read(ids))
            local = torch.rand(Q, 3, generator=gen).to(cuda_device)
            ids = tree(local, want_node_ids=True, world=False)[1]
            assert torch.equal(cache(local, world=False), cache.read(ids))
        rows = torch.randn(100, tree.data_dim, generator=gen).to(cuda_device)
        local = local[:100]
        cache.set(local, rows, world=False)
        same(cache(local, world=False)[-1:], held(rows[-1:], cache.group, INT8))


@pytest.mark.gpu
def test_cache_is_a_snapshot(cuda_device):
    tree = make_tree("SH4", cuda_device, refine=2)
    cache = svox.RecordCache(tree)
    points = torch.rand(300, 3, device=cuda_device)
    want = cache(points)
    with torch.no_grad():
        tree.data.data.zero_()
    tree.refine()
    assert torch.equal(cache(points), want)
    assert set(cache.state_dict()) == {"child", "offset", "invradius", "records", "_extra_state"}
    same_shape = svox.RecordCache(make_tree("SH4", cuda_device, refine=2))
    same_shape.write(torch.arange(50, device=cuda_device), torch.ones(50, 13, device=cuda_device))
    same_shape.load_state_dict(cache.state_dict())
    assert torch.equal(same_shape(points), want)
    kind = svox.RecordCache(make_tree("SH4", cuda_device, refine=2), dtype=E4M3)
    with pytest.raises(RuntimeError, match="record cache"):
        kind.load_state_dict(cache.state_dict())
    import copy
    twin = copy.deepcopy(cache)
    twin.set(points, want + 1)
    assert torch.equal(cache(points), want)
    assert cache(points[:0]).shape == (0, 13)
    cache.set(points[:0], want[:0])
    cache.write(torch.zeros(0, dtype=torch.int64, device=cuda_device), want[:0])
    # strides and other types
    wide = torch.rand(300, 5, device=cuda_device)
    assert torch.equal(cache(wide[:, 1:4]), cache(wide[:, 1:4].contiguous()))
    assert torch.equal(cache(wide[:, 1:4].double()), cache(wide[:, 1:4].contiguous()))
    rows = torch.randn(300, 26, device=cuda_device)[:, ::2]
    cache.set(points, rows)
    again = cache(points)
    cache.set(points, rows.double().contiguous())
    assert torch.equal(cache(points), again)


@pytest.mark.gpu
def test_ids_out_of_range(cuda_device):
    tree = make_tree("SH4", cuda_device, refine=1)
    cache = svox.RecordCache(tree)
    n = len(cache)
    before = cache.records.clone()
    ids = torch.tensor([0, -1, n - 1, n, 1 << 40, -(1 << 62)], device=cuda_device)
    csrc.device_status()
    out = cache.read(ids)
    assert csrc.device_status() == 9
    ok = torch.tensor([True, False, True, False, False, False], device=cuda_device)
    assert out[~ok].isnan().all() and torch.equal(out[ok], cache.read(ids[ok]))
    cache.write(ids, torch.ones(6, 13, device=cuda_device))
    assert csrc.device_status() == 9 and csrc.device_status() == 0
    rest = torch.ones(n, dtype=torch.bool, device=cuda_device)
    rest[ids[ok]] = False
    assert torch.equal(cache.records[rest], before[rest])
    assert (cache.read(ids[ok]) == 1).all() and (cache._owner == 0).all()


@pytest.mark.gpu
def test_streams_and_graphs(cuda_device):
    tree = make_tree("SH9", cuda_device, refine=3)
    cache = svox.RecordCache(tree)
    gen = torch.Generator().manual_seed(4)
    points = torch.rand(5000, 3, generator=gen).to(cuda_device)
    rows = torch.randn(5000, 28, generator=gen).to(cuda_device)

    def step():
        cache.set(points, rows)
        return cache(points, dtype=BF16)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            want = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(step(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held_out = step()
    rows *= 0.5
    points.copy_(points.flip(0))
    for _ in range(2):
        graph.replay()
    assert torch.equal(step(), held_out)
    assert (cache._owner == 0).all()


@pytest.mark.gpu
def test_refusals_gpu(cuda_device):
    tree = make_tree("SH4", cuda_device, refine=1)
    cache = svox.RecordCache(tree)
    points = torch.rand(5, 3, device=cuda_device)
    rows = torch.rand(5, 13, device=cuda_device)
    ids = torch.zeros(5, dtype=torch.int64, device=cuda_device)
    for call in (lambda: cache(points[:, :2]), lambda: cache(points.cpu()),
                 lambda: cache(points, dtype=torch.float64), lambda: cache.read(ids.int()),
                 lambda: cache.read(ids[None]), lambda: cache.read(ids.cpu()),
                 lambda: cache.set(points, rows[:, :5]), lambda: cache.set(points, rows[:4]),
                 lambda: cache.set(points, rows.cpu()), lambda: cache.write(ids, rows[:3]),
                 lambda: cache.write(ids, rows.clone().requires_grad_(True)),
                 lambda: svox.RecordCache(tree, dtype=torch.uint8),
                 lambda: svox.RecordCache(tree, group=0),
                 lambda: svox.RecordCache(svox.N3Tree(data_dim=1, device=cuda_device))):
        with pytest.raises(RuntimeError):
            call()


def test_refusals():
    tree = svox.N3Tree(data_format="SH4")
    with pytest.raises(RuntimeError, match="CUDA device"):
        svox.RecordCache(tree)
    with pytest.raises(RuntimeError, match="int8"):
        svox.RecordCache(tree, dtype=torch.float32)


def test_record_layout():
    """Codes, exponents and density; the sizes that the documents name."""
    assert [csrc.record_bytes(3 * b + 1, b) for b in (1, 4, 9, 16, 25)] == [8, 32, 32, 64, 80]
    assert csrc.record_bytes(4, 3) == 8 and csrc.record_bytes(2, 1) == 8
    for K, group in ((1, 1), (5, 0), (1025, 4)):
        with pytest.raises(RuntimeError):
            csrc.record_bytes(K, group)


def test_abi_refusals():
    import ctypes as C

    class Records(C.Structure):
        _fields_ = [("records", C.c_void_p), ("owner", C.c_void_p), ("child", C.c_void_p),
                    ("offset", C.c_void_p), ("scaling", C.c_void_p), ("M", C.c_int64),
                    ("N", C.c_int32), ("K", C.c_int32), ("group", C.c_int32),
                    ("code_type", C.c_int32)]

    lib = csrc.library()

    def read(points=None, ids=16, Q=4, out=None, kind=0, **k):
        r = Records(16, 16, 16, 16, 16, 1, 2, 4, 3, 0)
        for name, v in k.items():
            setattr(r, name, v)
        return lib.svoxb_records_read(C.byref(r), C.c_void_p(points), C.c_void_p(ids),
                                      C.c_int64(Q), C.c_void_p(out), C.c_int32(kind), None)

    assert read() == 1 and read(records=None) == 1 and read(points=16) == 4
    assert read(points=16, ids=None, child=None) == 1
    assert read(Q=-1) == 2 and read(K=1) == 2 and read(group=0) == 2 and read(N=1) == 2
    assert read(ids=None, Q=9) == 2                 # more rows than records
    assert read(kind=3) == 3 and read(code_type=2) == 3
    assert read(Q=1 << 32) == 8 and read(K=1025) == 8
    assert read(Q=0) == 0
    r = Records(16, None, 16, 16, 16, 1, 2, 4, 3, 0)
    assert lib.svoxb_records_write(C.byref(r), None, C.c_void_p(16), C.c_int64(4), C.c_void_p(16),
                                   C.c_int32(0), C.c_void_p(16), None) == 1     # no owner
    r.owner = 16
    assert lib.svoxb_records_write(C.byref(r), None, C.c_void_p(16), C.c_int64(4), C.c_void_p(16),
                                   C.c_int32(0), None, None) == 1               # no workspace


@pytest.mark.gpu
def test_a_refused_state_changes_nothing(cuda_device):
    """A cache's state is taken whole or not at all, on its own and as a part of another module."""
    kind = svox.RecordCache(make_tree("SH4", cuda_device, refine=2), dtype=E4M3)
    kind.invradius *= 0.5
    other = svox.RecordCache(make_tree("SH4", cuda_device, refine=2))
    larger = svox.RecordCache(make_tree("SH4", cuda_device, refine=3), dtype=E4M3)
    state = other.state_dict()
    unsaid = {k: v for k, v in kind.state_dict().items() if k != "_extra_state"}
    part = {k: v for k, v in kind.state_dict().items() if k != "child"}
    before = {k: v.clone() for k, v in kind.state_dict().items() if k != "_extra_state"}
    for bad in (state, larger.state_dict(), unsaid, part):
        bad = {k: torch.zeros_like(v) + 1 if k == "records" else v for k, v in bad.items()}
        for strict in (True, False):
            with pytest.raises(RuntimeError):
                kind.load_state_dict(bad, strict=strict)
            holder = torch.nn.ModuleDict({"cache": kind})
            with pytest.raises(RuntimeError):
                holder.load_state_dict({"cache." + k: v for k, v in bad.items()}, strict=strict)
            for k, v in before.items():
                assert torch.equal(kind.state_dict()[k], v), k
    # a state of something else without a word of the cache, and its own
    torch.nn.ModuleDict({"cache": kind}).load_state_dict({}, strict=False)
    twin = svox.RecordCache(make_tree("SH4", cuda_device, refine=2), dtype=E4M3)
    twin.write(torch.arange(50, device=cuda_device), torch.ones(50, 13, device=cuda_device))
    torch.nn.ModuleDict({"cache": twin}).load_state_dict(
        torch.nn.ModuleDict({"cache": kind}).state_dict())
    assert torch.equal(twin.read(), kind.read()) and torch.equal(twin.invradius, kind.invradius)


@pytest.mark.gpu
def test_views_of_negatives(cuda_device):
    """Points and values whose memory holds their negatives."""
    cache = svox.RecordCache(make_tree("SH4", cuda_device, refine=2))
    points = torch.rand(200, 3, device=cuda_device)
    rows = torch.randn(200, 13, device=cuda_device)
    cache.set(points, rows)
    want = cache(points)
    cache.set(points, rows + 1)
    view = torch._neg_view
    assert view(-points).is_neg()
    cache.set(view(-points), view(-rows))
    assert torch.equal(cache(points), want) and torch.equal(cache(view(-points)), want)
