"""The global gradient norm and clipping against plain 64-bit arithmetic.

Tolerances.  Runs of at most 32 squares are summed in fp32 (32 * 2^-24, and
the root halves it), everything above in fp64, and the norm is rounded to fp32
once: RTOL_NORM = 2e-6.  The factor adds a sum and a quotient, a clipped value
one product and one rounding to its type."""

import math

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from practice_cuda_b200 import _lib
from practice_cuda_b200.grad_clip import clip_grad_norm, clip_grad_norm_, grad_norm, join_norms
from tests._util import synthetic

gpu = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}
RTOL_NORM = 2e-6
EPS = 1e-6


def _tensors(sizes, dtypes, seed=0, std=1.0):
    return [synthetic((n,), std=std, outliers=n > 0, seed=seed + i, dtype=dtypes[i % len(dtypes)]).cuda() if n
            else torch.empty(0, device="cuda", dtype=dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def _norm64(tensors):
    return math.sqrt(sum(t.double().square().sum().item() for t in tensors))


def _check_clipped(got, before, factor):
    for g, b in zip(got, before):
        assert g.dtype == b.dtype and g.shape == b.shape
        if not g.numel():
            continue
        expected = b.double() * factor
        d = (g.double() - expected).abs()
        bound = (UNIT[g.dtype] + 3 * RTOL_NORM) * expected.abs() + TINY[g.dtype]
        assert bool((d <= bound).all()), f"{g.dtype} off by {d.max().item():.3e}"


SIZES = [
    [1],
    [7, 8, 9],
    [0, 5, 0, 17],
    [8191, 8192, 8193, 16384, 16385],
    [100003, 64, 3],
    [300] * 64,  # a full small table
    [300] * 65,  # the next table size
    [37] * 1000 + [1001, 5, 2049],  # more than one table
    [5_000_011],
]


@gpu
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (BF16, F32, F16)], ids=lambda d: "+".join(str(t)[6:] for t in d))
def test_norm_and_clip(sizes, dtypes):
    tensors = _tensors(sizes, dtypes, seed=len(sizes))
    before = [t.clone() for t in tensors]
    norm64 = _norm64(tensors)
    norm = grad_norm(tensors)
    assert norm.dtype == F32 and norm.ndim == 0
    assert abs(norm.item() - norm64) <= RTOL_NORM * norm64
    # into other tensors: the gradients stay
    max_norm = 0.37 * norm64
    out = [torch.full_like(t, 3.0) for t in tensors]
    got = clip_grad_norm(tensors, max_norm, out=out)
    assert torch.equal(got, norm) and all(torch.equal(t, b) for t, b in zip(tensors, before))
    factor = min(1.0, max_norm / (norm64 + EPS))
    _check_clipped(out, before, factor)
    # in place: the same values
    assert torch.equal(clip_grad_norm(tensors, max_norm), norm)
    assert all(torch.equal(t, o) for t, o in zip(tensors, out))
    # below the limit nothing changes, in place or not
    kept = [t.clone() for t in tensors]
    clip_grad_norm(tensors, 2 * norm64)
    clip_grad_norm(tensors, 2 * norm64, out=out)
    assert all(torch.equal(t, k) and torch.equal(o, k) for t, k, o in zip(tensors, kept, out))


@gpu
@pytest.mark.parametrize("sizes", SIZES[1:6], ids=lambda s: f"{len(s)}x{max(s)}")
def test_largest_magnitude(sizes):
    tensors = _tensors(sizes, (BF16, F32), seed=3)
    largest = max(t.abs().max().item() for t in tensors if t.numel())
    before = [t.clone() for t in tensors]
    norm = clip_grad_norm(tensors, 0.5 * largest, norm_type=math.inf)
    assert norm.item() == largest
    _check_clipped(tensors, before, min(1.0, 0.5 * largest / (largest + EPS)))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_offsets_that_are_not_16_byte_aligned(dtype):
    for a in range(9):
        for b in (0, 1, 5):
            base = synthetic((9000 + 32,), seed=a, dtype=dtype).cuda()
            target = torch.zeros(9000 + 32, device="cuda", dtype=dtype)
            for n in (1, 6, 16, 8191, 9000):
                g, o = base[a : a + n], target[b : b + n]
                norm64 = _norm64([g])
                norm = clip_grad_norm([g], 0.5 * norm64, out=[o])
                assert abs(norm.item() - norm64) <= RTOL_NORM * norm64
                _check_clipped([o], [g], min(1.0, 0.5 * norm64 / (norm64 + EPS)))
                assert int(target[b + n :].count_nonzero()) == 0 and int(target[:b].count_nonzero()) == 0
                target.zero_()


@gpu
def test_strides():
    base = synthetic((64, 96), seed=5).cuda()
    views = [base.t(), base[:, ::2], base[3:9, 5:77], base.view(8, 8, 96).permute(2, 0, 1)]
    for v in views:
        norm64 = _norm64([v])
        assert abs(grad_norm([v]).item() - norm64) <= RTOL_NORM * norm64
        before = v.clone()
        rest = base.clone()
        clip_grad_norm([v], 0.5 * norm64)
        _check_clipped([v], [before], 0.5 * norm64 / (norm64 + EPS))
        changed = torch.zeros_like(base, dtype=torch.bool)
        torch.as_strided(changed, v.shape, v.stride(), v.storage_offset()).fill_(True)
        assert torch.equal(base[~changed], rest[~changed])
        base.copy_(rest)
    out = torch.empty(96, 64, device="cuda", dtype=BF16).t()  # another order than its gradient's
    norm64 = _norm64([base])
    clip_grad_norm([base], 0.5 * norm64, out=[out])
    _check_clipped([out], [base], 0.5 * norm64 / (norm64 + EPS))
    expanded = base[:1].expand(64, 96)
    assert abs(grad_norm([expanded]).item() - _norm64([expanded])) <= RTOL_NORM * _norm64([expanded])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_range_of_the_squares(dtype):
    big = torch.full((5000,), 3e30, device="cuda", dtype=dtype)  # its square is beyond fp32
    expected = _norm64([big])
    assert abs(grad_norm([big]).item() - expected) <= RTOL_NORM * expected
    before = big.clone()
    clip_grad_norm([big], 1.0)
    _check_clipped([big], [before], 1.0 / expected)


@gpu
def test_zero_and_non_finite_gradients():
    zero = torch.zeros(1000, device="cuda")
    assert clip_grad_norm([zero], 1.0).item() == 0.0 and int(zero.count_nonzero()) == 0
    assert clip_grad_norm([zero], 0.0, eps=0.0).item() == 0.0 and int(zero.count_nonzero()) == 0
    for bad, norm_type in ((math.nan, 2.0), (math.inf, 2.0), (math.nan, math.inf), (math.inf, math.inf)):
        g = [torch.ones(3000, device="cuda"), torch.ones(100, device="cuda", dtype=BF16)]
        g[0][2999] = bad
        kept = [t.clone() for t in g]
        with pytest.raises(RuntimeError, match="norm is"):
            clip_grad_norm(g, 1.0, norm_type=norm_type, error_if_nonfinite=True)
        assert torch.equal(g[0][:2999], kept[0][:2999]) and torch.equal(g[1], kept[1])
        norm = clip_grad_norm(g, 1.0, norm_type=norm_type)
        if math.isnan(bad):
            assert math.isnan(norm.item()) and bool(torch.isnan(g[1]).all())
        else:
            assert norm.item() == math.inf and int(g[1].count_nonzero()) == 0 and math.isnan(g[0][2999].item())
    fine = [torch.ones(10, device="cuda")]
    clip_grad_norm(fine, 1.0, error_if_nonfinite=True)
    _check_clipped(fine, [torch.ones(10, device="cuda")], 1.0 / (math.sqrt(10) + EPS))


@gpu
def test_parameters_and_repeatability():
    model = torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.Linear(65, 7)).cuda()
    model[1].bias.requires_grad_(False)
    model(torch.randn(12, 33, device="cuda")).square().sum().backward()
    grads = [p.grad.clone() for p in model.parameters() if p.grad is not None]
    norm64 = _norm64(grads)
    norm = clip_grad_norm_(model.parameters(), 0.1)
    assert abs(norm.item() - norm64) <= RTOL_NORM * norm64
    _check_clipped([p.grad for p in model.parameters() if p.grad is not None], grads, 0.1 / (norm64 + EPS))
    many = _tensors([40009] * 70, (BF16, F32), seed=9)
    assert len({grad_norm(many).item() for _ in range(5)}) == 1
    assert clip_grad_norm_([torch.nn.Parameter(torch.ones(3))], 1.0).item() == 0.0  # no gradients


@gpu
def test_clipping_inside_a_graph_is_seen():
    x = torch.ones(64, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    loss = (g * g).sum()  # keeps g
    clip_grad_norm([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@gpu
def test_stream_and_graph():
    g = _tensors([4097, 100], (F32,), seed=11)
    before = [t.clone() for t in g]
    out = [torch.empty_like(t) for t in g]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        clip_grad_norm(g, 1.0, out=out)
    stream.synchronize()
    _check_clipped(out, before, 1.0 / (_norm64(before) + EPS))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm(g, 1.0, out=out)
    for t in g:
        t.mul_(4.0)
    graph.replay()
    assert abs(norm.item() - 4 * _norm64(before)) <= RTOL_NORM * 4 * _norm64(before)
    _check_clipped(out, before, 4.0 / (4 * _norm64(before) + EPS))


@gpu
def test_refusals():
    g = torch.ones(8, device="cuda")
    for bad in (
        lambda: clip_grad_norm([g], -1.0),
        lambda: clip_grad_norm([g], math.nan),
        lambda: clip_grad_norm([g], 1.0, norm_type=1.0),
        lambda: clip_grad_norm([], 1.0),
        lambda: clip_grad_norm([g.int()], 1.0),
        lambda: clip_grad_norm([g], 1.0, out=[]),
        lambda: clip_grad_norm([g], 1.0, out=[g[:4]]),
        lambda: clip_grad_norm([g], 1.0, out=[g.half()]),
        lambda: clip_grad_norm([g, g.cpu()], 1.0),
        lambda: clip_grad_norm([g[:1].expand(8)], 1.0),
        lambda: grad_norm([g], norm_type="two"),
    ):
        with pytest.raises(ValueError):
            bad()


def test_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        grad_norm([torch.ones(3)])


def _join_worker(rank, path, results):
    dist.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=2)
    own = torch.tensor([3.0, 4.0][rank])
    got = [join_norms(own, 2.0, dist.group.WORLD).item(), join_norms(own, math.inf, dist.group.WORLD).item()]
    bad = torch.tensor([math.nan, 4.0][rank])
    got += [join_norms(bad, 2.0, dist.group.WORLD).item(), join_norms(bad, math.inf, dist.group.WORLD).item()]
    far = torch.tensor([3e30, 4e30][rank])
    got.append(join_norms(far, 2.0, dist.group.WORLD).item())
    results[rank] = got
    dist.destroy_process_group()


def test_norms_of_several_processes(tmp_path):
    with mp.Manager() as manager:
        results = manager.dict()
        mp.spawn(_join_worker, args=(str(tmp_path / "store"), results), nprocs=2)
        for rank in range(2):
            l2, largest, nan2, nan_inf, far = results[rank]
            assert l2 == 5.0 and largest == 4.0 and math.isnan(nan2) and math.isnan(nan_inf)
            assert abs(far - 5e30) <= RTOL_NORM * 5e30


def test_entry_points_reject_bad_arguments_without_gpu():
    import ctypes

    lib = _lib.lib()
    one = (ctypes.c_uint64 * 1)(16)
    size = (ctypes.c_int64 * 1)(4)

    def clip(numel=4, dtype=0, norm_type=0, max_norm=1.0, pointer=16, norm=16, nbytes=1 << 20, count=1):
        one[0], size[0] = pointer, numel
        kind = (ctypes.c_int * 1)(dtype)
        return lib.pcb_grad_clip(ctypes.addressof(one), ctypes.addressof(one), ctypes.addressof(size),
                                 ctypes.addressof(kind), count, norm_type, max_norm, EPS, norm, 16, nbytes, None)

    for kwargs in ({"numel": -1}, {"dtype": 3}, {"norm_type": 2}, {"max_norm": -1.0}, {"max_norm": math.nan},
                   {"pointer": 0}, {"pointer": 17}, {"norm": None}, {"nbytes": 0}, {"count": -1}):
        assert clip(**kwargs) == _lib.PCB_ERR_INVALID, kwargs
    assert lib.pcb_grad_norm(None, None, None, 1, 0, 16, 16, 1 << 20, None) == _lib.PCB_ERR_INVALID


def test_overlapping_tensors_are_refused_without_gpu():
    """Two CTAs would scale the same elements at once."""
    import ctypes

    lib = _lib.lib()

    def status(entry, grads, out, numel, dtypes=None):
        count = len(grads)
        pointers, targets = (ctypes.c_uint64 * count)(*grads), (ctypes.c_uint64 * count)(*out)
        sizes, kinds = (ctypes.c_int64 * count)(*numel), (ctypes.c_int * count)(*(dtypes or [0] * count))
        table = (ctypes.addressof(pointers), ctypes.addressof(targets), ctypes.addressof(sizes), ctypes.addressof(kinds))
        if entry == "clip":  # a norm that is missing is refused too, but later
            return lib.pcb_grad_clip(*table, count, 0, 1.0, EPS, None, None, 0, None), lib.pcb_last_error_text().decode()
        return lib.pcb_grad_scale(*table, count, None, 1.0, EPS, None), lib.pcb_last_error_text().decode()

    bad = [
        ([64, 64], [64, 64], [4, 4]),  # one tensor twice
        ([256, 64, 256], [256, 64, 256], [4, 4, 4]),
        ([64, 72], [64, 72], [4, 4]),  # 16 bytes from 64 on, and from 72 on
        ([64, 128], [128, 64], [4, 4]),  # outputs changed over
        ([64, 128], [256, 264], [4, 4]),  # outputs that overlap
        ([64], [68], [4]),  # an output that is moved by less than its length
        ([64, 80, 512], [64, 80, 92], [4, 4, 4]),  # an output in another gradient
    ]
    good = [
        ([64, 80], [64, 80], [4, 4]),  # neighbours
        ([80, 64], [80, 64], [4, 4]),
        ([64, 64], [256, 512], [4, 4]),  # one gradient into two outputs
        ([64, 64], [64, 64], [4, 0]),  # an empty tensor
        ([64, 128], [256, 272], [4, 4]),
        ([64], [80], [4]),
        ([64, 80, 512], [64, 80, 96], [4, 4, 4]),
    ]
    for entry in ("clip", "scale"):
        for case in bad:
            code, text = status(entry, *case)
            assert code == _lib.PCB_ERR_INVALID and "overlap" in text, case
        for case in good:
            assert "overlap" not in status(entry, *case)[1], case
        assert "overlap" in status(entry, [64, 72], [64, 72], [4, 4], [0, 0])[1]
        assert "overlap" not in status(entry, [64, 72], [64, 72], [4, 4], [1, 1])[1]  # 8 bytes each


@gpu
def test_overlapping_tensors_are_refused():
    g = torch.arange(1.0, 101.0, device="cuda").view(10, 10)
    kept, other = g.clone(), torch.empty_like(g)
    parameter = torch.nn.Parameter(torch.zeros(10, 10, device="cuda"))
    parameter.grad = g
    for bad in (
        lambda: clip_grad_norm([g, g], 1.0),
        lambda: clip_grad_norm([g, g], 1.0, error_if_nonfinite=True),
        lambda: clip_grad_norm([g[:6], g[5:]], 1.0),
        lambda: clip_grad_norm([g, other], 1.0, out=[other, g]),
        lambda: clip_grad_norm([g, kept], 1.0, out=[other, other]),
        lambda: clip_grad_norm([g[:, ::2], g[:, ::2]], 1.0),  # strided ones
        lambda: clip_grad_norm_([parameter, parameter], 1.0),
    ):
        with pytest.raises(ValueError, match="overlap"):
            bad()
    assert torch.equal(g, kept)
    norm64 = _norm64([kept])
    # Neighbours, columns that take turns, and a gradient that is read twice are fine.
    clip_grad_norm([g[:5], g[5:]], 0.5 * norm64)
    _check_clipped([g], [kept], 0.5 * norm64 / (norm64 + EPS))
    g.copy_(kept)
    clip_grad_norm([g[:, ::2], g[:, 1::2]], 0.5 * norm64)
    _check_clipped([g], [kept], 0.5 * norm64 / (norm64 + EPS))
    twice = [torch.empty_like(g), torch.empty_like(g)]
    clip_grad_norm([kept, kept], norm64, out=twice)
    _check_clipped(twice, [kept, kept], norm64 / (math.sqrt(2.0) * norm64 + EPS))


@gpu
def test_clipping_what_a_graph_has_saved_is_seen():
    """Gradients do not require a gradient themselves, but a graph may hold them."""
    w = torch.ones(64, device="cuda", requires_grad=True)
    plain = lambda: torch.full((8, 8), 3.0, device="cuda")
    targets = {
        "in place": lambda g: clip_grad_norm([g], 0.1),
        "in place, not finite": lambda g: clip_grad_norm([g], 0.1, error_if_nonfinite=True),
        "an output": lambda g: clip_grad_norm([plain()], 0.1, out=[g]),
        "detached": lambda g: clip_grad_norm([g.detach()], 0.1),
        "a view": lambda g: clip_grad_norm([g[2:5]], 0.1),
        "columns": lambda g: clip_grad_norm([g[:, 2:5]], 0.1),
        "beside a strided one": lambda g: clip_grad_norm([plain()[:, ::2], g], 0.1),
    }
    for name, clip in targets.items():
        g = plain()
        loss = (w * g.view(64)).sum()  # keeps g
        version = g._version
        clip(g)
        assert g._version > version, name
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    # What is read alone keeps its version.
    g, out = plain(), plain()
    version = g._version
    clip_grad_norm([g], 0.1, out=[out])
    grad_norm([g])
    assert g._version == version
    with torch.inference_mode():
        clip_grad_norm([plain()], 0.1)


def test_clipping_sharded_gradients_is_seen_without_gpu(tmp_path, monkeypatch):
    """The DTensor that holds a clipped shard counts the change too."""
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Shard, distribute_tensor

    from practice_cuda_b200 import grad_clip

    monkeypatch.setattr(grad_clip, "clip_grad_norm", lambda tensors, *args, **kwargs: torch.ones(()))
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cpu", (1,))
        parameter = torch.nn.Parameter(distribute_tensor(torch.ones(4, 2), mesh, [Shard(0)]))
        parameter.grad = distribute_tensor(torch.full((4, 2), 3.0), mesh, [Shard(0)])
        version = parameter.grad._version
        grad_clip.clip_grad_norm_([parameter], 0.1)
        assert parameter.grad._version > version
    finally:
        dist.destroy_process_group()


@gpu
@pytest.mark.parametrize("value", [1e-18, 1e-20, 1e-23, 1e-30, 1e-36])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_squares_below_the_range_of_fp32(value, dtype):
    """Gradients whose squares are subnormal or nothing in fp32: the norm has the same accuracy."""
    for sizes in ([5000], [1], [7, 8193, 40]):
        small = [synthetic((n,), std=value, seed=n, dtype=dtype).cuda() for n in sizes]
        expected = _norm64(small)
        assert abs(grad_norm(small).item() - expected) <= RTOL_NORM * expected
        before = [t.clone() for t in small]
        norm = clip_grad_norm(small, 0.5 * expected, eps=0.0)
        assert abs(norm.item() - expected) <= RTOL_NORM * expected
        _check_clipped(small, before, 0.5)
    # Large ones beside them, and zeros.
    mixed = [torch.full((300,), value, device="cuda", dtype=dtype), torch.zeros(5000, device="cuda", dtype=dtype),
             torch.ones(3, device="cuda", dtype=dtype)]
    assert abs(grad_norm(mixed).item() - _norm64(mixed)) <= RTOL_NORM * _norm64(mixed)
    mixed.pop()
    assert abs(grad_norm(mixed).item() - _norm64(mixed)) <= RTOL_NORM * _norm64(mixed)
