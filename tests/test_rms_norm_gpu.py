"""The root-mean-square norm with the residual's addition and an FP8 output,
against plain 64-bit arithmetic.

Tolerances.  fp32 arithmetic: a sum of squares is a tree of at most a few
dozen sequential roundings (2^-24 each), its root halves them, and y adds
three products: RTOL32 = 4e-6 covers 64 of them.  A value rounded once to its
type is off by at most half a unit in the last place (UNIT).  An FP8 value is
the nearest grid point unless the exact quotient lies within RTOL32 of a tie,
so it may be one grid step off, which happens to about 2 * RTOL32 / 2^-4 of
all values at most (QUANT_FLIPS, with room for small counts)."""

import pytest
import torch

from practice_cuda_b200 import _lib
from practice_cuda_b200.rms_norm import rms_norm, rms_norm_backward, rms_norm_quant
from tests._util import E4M3, E5M2, synthetic

gpu = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}  # half the smallest subnormal
RTOL32 = 4e-6
QUANT_FLIPS = 1e-3
FP8_MAX = {E4M3: 448.0, E5M2: 57344.0}
EPS = 1e-5

SHAPES = [
    (1, 4096),  # one token
    (3, 64), (9, 128), (8, 256), (17, 512), (5, 1000), (4, 2048), (7, 2056), (3, 4096), (2, 7168), (2, 8192),
    (2, 8200), (3, 16384), (2, 20000), (1, 32768), (1, 40000),  # widths of every lane count
    (5, 1), (4, 7), (6, 129), (3, 1021), (2, 5003),  # odd widths: element by element
    (2000, 264),
]


def _inputs(rows, dim, dtype, seed, residual=True):
    x = synthetic((rows, dim), outliers=True, seed=seed, dtype=dtype).cuda()
    r = synthetic((rows, dim), outliers=True, seed=seed + 1, dtype=dtype).cuda() if residual else None
    w = (1.0 + 0.1 * synthetic((dim,), seed=seed + 2, dtype=F32)).to(dtype).cuda()
    return x, r, w


def _reference(x, w, r, eps=EPS):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    h64 = h.double()
    rstd = 1.0 / torch.sqrt(h64.square().mean(-1) + eps)
    return h, h64 * rstd[..., None] * w.double(), rstd


def _close(actual, expected, rtol, atol, what):
    d = (actual.double() - expected).abs()
    bound = rtol * expected.abs() + atol
    assert bool((d <= bound).all()), f"{what}: off by {d.max().item():.3e}, worst ratio {(d / bound).max().item():.2f}"


def _check_quant(result, y64, quant, fp8, pow2, what):
    rows, dim = y64.shape
    block = 128 if quant == "block" else dim
    blocks = -(-dim // block)
    padded = torch.nn.functional.pad(y64, (0, blocks * block - dim)).view(rows, blocks, block)
    amax = padded.abs().amax(2).clamp_min(1e-12)
    scale = amax / FP8_MAX[fp8]
    if pow2:
        scale = torch.exp2(torch.ceil(torch.log2(scale)))
    got = result.dequant_scale.view(rows, blocks).double()
    _close(got, scale, RTOL32, 0.0, f"{what} scale")
    spread = got.repeat_interleave(block, 1)[:, :dim]
    expected = (y64 / spread).clamp(-FP8_MAX[fp8], FP8_MAX[fp8]).to(fp8)
    q = result.tensor
    assert q.dtype == fp8 and tuple(q.shape) == (rows, dim)
    a, e = q.view(torch.uint8).int(), expected.view(torch.uint8).int()
    off = (a - e).abs()
    off = torch.where(((a ^ e) == 128) & (q.double() == 0), 0, off)  # a zero's sign
    assert int(off.max()) <= 1, f"{what}: {int((off > 1).sum())} FP8 values are more than one grid step off"
    assert int((off > 0).sum()) <= max(2, QUANT_FLIPS * off.numel()), f"{what}: {int((off > 0).sum())} values flipped"


def _check_forward(x, r, w, quant, fp8, pow2=False, keep=True, what=""):
    res = rms_norm_quant(x, w, r, eps=EPS, quant=quant, fp8_dtype=fp8, pow2_scales=pow2, return_y=keep)
    h, y64, rstd = _reference(x, w, r)
    assert torch.equal(res.residual, h), f"{what} residual"
    _close(res.rstd, rstd, RTOL32, 0.0, f"{what} rstd")
    if keep or quant is None:
        _close(res.y, y64, UNIT[x.dtype] * (1 + 1e-3) + RTOL32, TINY[x.dtype], f"{what} y")
    else:
        assert res.y is None
    if quant is None:
        assert res.quant is None
    else:
        _check_quant(res.quant, y64, quant, fp8, pow2, what)
    return res


@gpu
@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_forward_widths(rows, dim, dtype):
    x, r, w = _inputs(rows, dim, dtype, seed=rows + dim)
    _check_forward(x, r, w, "block", E4M3, what="block")
    _check_forward(x, None, w, "row", E5M2, keep=False, what="row")
    _check_forward(x, r, w.float(), None, E4M3, what="y alone, fp32 weight")


@gpu
@pytest.mark.parametrize("rows,dim", [(5, 511), (4, 513), (3, 2047), (3, 2049), (2, 4095), (2, 4097), (3, 6143),
                                      (2, 6145), (2, 8191), (2, 8193), (2, 16383), (1300, 2051)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_forward_odd_widths(rows, dim, dtype):
    x, r, w = _inputs(rows, dim, dtype, seed=rows + dim)
    for residual in (r, None):
        _check_forward(x, residual, w, "block", E4M3, what="block")
        _check_forward(x, residual, w, "row", E4M3, what="row")
        _check_forward(x, residual, w.float(), None, E4M3, what="y alone, fp32 weight")


@gpu
@pytest.mark.parametrize("dim", [4101, 8195])
def test_forward_odd_zero_rows_and_non_finite_values(dim):
    x, _, w = _inputs(5, dim, BF16, seed=3)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    for residual in (None, torch.zeros_like(x)):
        res = rms_norm_quant(x, w, residual, eps=EPS, return_y=True)
        assert torch.equal(res.y[1], torch.zeros_like(res.y[1]))
        assert torch.equal(res.quant.tensor[1].float(), torch.zeros(dim, device="cuda"))
        assert bool(torch.isnan(res.y[3]).all())
        assert bool(torch.isnan(res.y[2, 5])) and torch.equal(res.y[2, 6:].float(),
                                                              torch.zeros(dim - 6, device="cuda"))
        good = [0, 4]
        _check_forward(x[good], None if residual is None else residual[good], w, "block", E4M3, what="rows beside them")


@gpu
@pytest.mark.parametrize("rows,dim", [(5, 512), (3, 4096), (9, 515), (2, 16392), (2, 20001)])
@pytest.mark.parametrize("dtype,wdtype", [(BF16, F16), (F16, BF16), (F32, BF16), (F32, F16), (F16, F32)])
def test_weights_of_another_type(rows, dim, dtype, wdtype):
    x, r, w = _inputs(rows, dim, dtype, seed=rows * dim)
    w = w.to(wdtype)
    _check_forward(x, r, w, "block", E4M3, what="block")
    res = _check_forward(x, None, w, "row", E4M3, what="row")
    dx, dw = rms_norm_backward(r, x, w, res.rstd)
    dx64, dw64, dx_terms, dw_terms = _backward_reference(r, x, w, res.rstd, None)
    _close(dx, dx64, UNIT[dtype] * (1 + 1e-3), TINY[dtype] + RTOL32 * dx_terms, "dx")
    _close(dw, dw64, UNIT[wdtype] * (1 + 1e-3), TINY[wdtype] + RTOL32 * dw_terms, "dw")


@gpu
@pytest.mark.parametrize("dim", [256, 1000, 129])
@pytest.mark.parametrize("fp8", [E4M3, E5M2])
def test_forward_power_of_two_scales(dim, fp8):
    x, r, w = _inputs(33, dim, BF16, seed=dim)
    res = _check_forward(x, r, w, "block", fp8, pow2=True, what="pow2")
    assert res.quant.meta["scale_format"] == "e8m0"
    mantissa = res.quant.dequant_scale.view(torch.int32) & 0x7FFFFF
    assert int(mantissa.max()) == 0


@gpu
@pytest.mark.parametrize("dim", [512, 515])
def test_forward_zero_rows_and_non_finite_values(dim):
    x, r, w = _inputs(6, dim, BF16, seed=3)
    x[1] = 0
    r[1] = 0  # a row of zeros: y is zero and the scale is that of quant_eps
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    res = rms_norm_quant(x, w, r, eps=EPS, return_y=True)
    assert torch.equal(res.y[1], torch.zeros_like(res.y[1]))
    assert torch.equal(res.quant.tensor[1].float(), torch.zeros(dim, device="cuda"))
    _close(res.quant.dequant_scale[1], torch.full_like(res.quant.dequant_scale[1], 1e-12 / 448.0).double(), RTOL32, 0.0,
           "zero row scale")
    assert bool(torch.isnan(res.y[3]).all())
    # inf / inf at the infinity, 0 elsewhere
    assert bool(torch.isnan(res.y[2, 5])) and torch.equal(res.y[2, 6:].float(), torch.zeros(dim - 6, device="cuda"))
    good = [0, 4, 5]
    _check_forward(x[good], r[good], w, "block", E4M3, what="rows beside them")


@gpu
def test_forward_views_strides_and_alignment():
    base = synthetic((6, 3 * 256 + 5), seed=9).cuda()
    w = synthetic((256,), seed=10).cuda()
    for start in (0, 256, 3, 517):  # 16-byte aligned rows or not
        x = base[:, start : start + 256]
        _check_forward(x, x, w, "block", E4M3, what=f"slice at {start}")
    x3 = synthetic((2, 5, 256), seed=11).cuda()
    res = rms_norm_quant(x3, w, x3, eps=EPS, return_y=True)
    assert res.y.shape == x3.shape and res.residual.shape == x3.shape and res.rstd.shape == (10,)
    flat = rms_norm_quant(x3.view(10, 256), w, x3.view(10, 256), eps=EPS, return_y=True)
    assert torch.equal(res.y.view(10, 256), flat.y)
    t = synthetic((256, 12), seed=12).cuda().t()  # rows not contiguous
    _check_forward(t, None, w, "row", E4M3, what="transposed")
    strided_w = synthetic((512,), seed=13).cuda()[::2]
    _check_forward(x3.view(10, 256), None, strided_w, "block", E4M3, what="strided weight")
    one = synthetic((256,), seed=14).cuda()
    assert torch.equal(rms_norm_quant(one, w, eps=EPS, return_y=True).y,
                       rms_norm_quant(one[None], w, eps=EPS, return_y=True).y[0])


@gpu
def test_no_rows():
    w = torch.ones(64, device="cuda", dtype=BF16)
    x = torch.empty((0, 64), device="cuda", dtype=BF16)
    res = rms_norm_quant(x, w, x)
    assert res.quant.tensor.shape == (0, 64) and res.quant.dequant_scale.shape == (0, 1) and res.rstd.shape == (0,)
    dx, dw = rms_norm_backward(x, x, w, res.rstd)
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


def _backward_reference(dy, h, w, rstd, dh):
    dy, h, w = dy.double(), h.double(), w.double()
    n = h * rstd.double()[:, None]
    wdy = w * dy
    dx = rstd.double()[:, None] * (wdy - n * (n * wdy).mean(1, keepdim=True))
    terms = rstd.double()[:, None] * (wdy.abs() + n.abs() * (n * wdy).abs().mean(1, keepdim=True))
    if dh is not None:
        dx, terms = dx + dh.double(), terms + dh.double().abs()
    return dx, (dy * n).sum(0), terms, (dy * n).abs().sum(0)


@gpu
@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (F16, F32), (F32, F32)])
def test_backward_widths(rows, dim, dtype, wdtype):
    h, dh, w = _inputs(rows, dim, dtype, seed=2 * rows + dim)
    w = w.to(wdtype)
    dy = synthetic((rows, dim), std=0.1, seed=5, dtype=dtype).cuda()
    rstd = (h.float().square().mean(1) + EPS).rsqrt()
    for extra in (dh, None):
        dx, dw = rms_norm_backward(dy, h, w, rstd, dresidual=extra)
        dx64, dw64, dx_terms, dw_terms = _backward_reference(dy, h, w, rstd, extra)
        # fp32 sums: RTOL32 of the sum of the terms' magnitudes, then one rounding.
        _close(dx, dx64, UNIT[dtype] * (1 + 1e-3), TINY[dtype] + RTOL32 * dx_terms, "dx")
        _close(dw, dw64, UNIT[wdtype] * (1 + 1e-3), TINY[wdtype] + RTOL32 * dw_terms, "dw")
        again = rms_norm_backward(dy, h, w, rstd, dresidual=extra)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)  # a fixed order of summation


@gpu
@pytest.mark.parametrize("rows,dim", [(1024, 4096), (4000, 72), (700, 1021)])
def test_backward_many_rows(rows, dim):
    h, dh, w = _inputs(rows, dim, BF16, seed=7)
    dy = synthetic((rows, dim), std=0.1, seed=8).cuda()
    rstd = (h.float().square().mean(1) + EPS).rsqrt()
    dx, dw = rms_norm_backward(dy, h, w.float(), rstd, dresidual=dh)
    dx64, dw64, dx_terms, dw_terms = _backward_reference(dy, h, w, rstd, dh)
    _close(dx, dx64, UNIT[BF16] * (1 + 1e-3), RTOL32 * dx_terms, "dx")
    _close(dw, dw64, UNIT[F32], RTOL32 * dw_terms, "dw")


@gpu
@pytest.mark.parametrize("rows,dim", [(700, 8200), (450, 10240), (297, 16384), (149, 12296), (300, 8192), (300, 16392),
                                      (300, 4099), (150, 8191), (297, 8193), (149, 16383), (20, 16385)])
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (F16, F32), (F32, F32)])
def test_backward_many_wide_rows(rows, dim, dtype, wdtype):
    h, dh, w = _inputs(rows, dim, dtype, seed=rows + dim)
    w = w.to(wdtype)
    wide = synthetic((rows, dim + 24), std=0.1, seed=8, dtype=dtype).cuda()
    dy = wide[:, 8 : 8 + dim]  # rows of another stride
    rstd = (h.float().square().mean(1) + EPS).rsqrt()
    for extra in (dh, None):
        dx, dw = rms_norm_backward(dy, h, w, rstd, dresidual=extra)
        dx64, dw64, dx_terms, dw_terms = _backward_reference(dy, h, w, rstd, extra)
        _close(dx, dx64, UNIT[dtype] * (1 + 1e-3), TINY[dtype] + RTOL32 * dx_terms, "dx")
        _close(dw, dw64, UNIT[wdtype] * (1 + 1e-3), TINY[wdtype] + RTOL32 * dw_terms, "dw")
        again = rms_norm_backward(dy, h, w, rstd, dresidual=extra)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@gpu
def test_backward_strides_and_alignment():
    dim = 256
    base = synthetic((5, 3 * dim + 7), seed=21, dtype=F32).cuda()
    w = synthetic((dim,), seed=22, dtype=F32).cuda()
    for at in ((0, dim, 2 * dim), (1, dim + 3, 2 * dim + 6)):
        dy, h, dh = (base[:, a : a + dim] for a in at)
        rstd = (h.square().mean(1) + EPS).rsqrt()
        dx, dw = rms_norm_backward(dy, h, w, rstd, dresidual=dh)
        dx64, dw64, dx_terms, dw_terms = _backward_reference(dy, h, w, rstd, dh)
        _close(dx, dx64, UNIT[F32], RTOL32 * dx_terms, "dx")
        _close(dw, dw64, UNIT[F32], RTOL32 * dw_terms, "dw")


@gpu
@pytest.mark.parametrize("dim", [264, 131])
def test_gradient_against_differences(dim):
    """Central differences of L = <y, a> + <h, b> along random directions.

    fp32 outputs summed in 64 bits: with a step of 1e-2 the cubic term is
    below 1e-4 of the derivative's scale and rounding adds about
    6e-8 * sqrt(values) * |a| / 1e-2; 2e-3 of the product of the norms covers
    both."""
    rows = 4
    x = synthetic((rows, dim), seed=31, dtype=F32).cuda().requires_grad_()
    r = synthetic((rows, dim), seed=32, dtype=F32).cuda().requires_grad_()
    w = synthetic((dim,), seed=33, dtype=F32).cuda().requires_grad_()
    a = synthetic((rows, dim), seed=34, dtype=F32).cuda()
    b = synthetic((rows, dim), seed=35, dtype=F32).cuda()

    def value(x, r, w):
        y, h, _ = rms_norm(x, w, r, eps=EPS)
        return (y.double() * a.double()).sum() + (h.double() * b.double()).sum()

    grads = torch.autograd.grad(value(x, r, w), (x, r, w))
    step = 1e-2
    for k, t in enumerate((x, r, w)):
        v = synthetic(tuple(t.shape), seed=40 + k, dtype=F32).cuda()
        v /= v.norm()
        with torch.no_grad():
            plus = [p + step * v if i == k else p for i, p in enumerate((x, r, w))]
            minus = [p - step * v if i == k else p for i, p in enumerate((x, r, w))]
            slope = (value(*plus) - value(*minus)) / (2 * step)
        assert abs((grads[k].double() * v.double()).sum() - slope).item() <= 2e-3 * grads[k].norm().item()


@gpu
def test_autograd_shapes_and_unused_outputs():
    x = synthetic((2, 3, 128), seed=51).cuda().requires_grad_()
    r = synthetic((2, 3, 128), seed=52).cuda().requires_grad_()
    w = torch.ones(128, device="cuda", dtype=F32).requires_grad_()
    y, h, q = rms_norm(x, w, r, quant="block")
    assert q.tensor.shape == (6, 128) and not q.tensor.requires_grad and y.shape == x.shape
    gx, gr = torch.autograd.grad(h.sum(), (x, r), retain_graph=True)  # h alone
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gr, gx)
    gx, gr, gw = torch.autograd.grad(y.sum(), (x, r, w))  # y alone
    assert gw.dtype == F32 and torch.equal(gx, gr)
    y2, h2, q2 = rms_norm(x, w)
    assert h2 is x and q2 is None
    assert torch.autograd.grad(y2.sum(), x)[0].shape == x.shape


@gpu
def test_runs_on_the_current_stream():
    x, r, w = _inputs(64, 512, BF16, seed=61)
    expected = rms_norm_quant(x, w, r, return_y=True).y
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = rms_norm_quant(x, w, r, return_y=True).y
    stream.synchronize()
    assert torch.equal(got, expected)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = rms_norm_quant(x, w, r, return_y=True).y
    x.copy_(x.flip(0))
    r.copy_(r.flip(0))
    graph.replay()
    assert torch.equal(captured, expected.flip(0))


@gpu
def test_refusals():
    x = torch.ones((4, 64), device="cuda", dtype=BF16)
    w = torch.ones(64, device="cuda", dtype=BF16)
    rstd = torch.ones(4, device="cuda")
    for bad in (
        lambda: rms_norm_quant(x, w[:32]),
        lambda: rms_norm_quant(x, w.int()),
        lambda: rms_norm_quant(x.int(), w),
        lambda: rms_norm_quant(x, w, x[:2]),
        lambda: rms_norm_quant(x, w, x.float()),
        lambda: rms_norm_quant(x, w, quant="tensor"),
        lambda: rms_norm_quant(x, w, quant="row", pow2_scales=True),
        lambda: rms_norm_quant(x, w, fp8_dtype=BF16),
        lambda: rms_norm_quant(x, w.cpu()),
        lambda: rms_norm_quant(x[:, :0], w[:0]),
        lambda: rms_norm_backward(x, x, w, rstd[:2]),
        lambda: rms_norm_backward(x, x, w, rstd.half()),
        lambda: rms_norm_backward(x.float(), x, w, rstd),
        lambda: rms_norm_backward(x, x, w, rstd, dresidual=x[:1]),
    ):
        with pytest.raises(ValueError):
            bad()


def test_refuses_cpu_tensors():
    x = torch.ones((4, 64))
    with pytest.raises(ValueError, match="CUDA"):
        rms_norm_quant(x, torch.ones(64))
    with pytest.raises(ValueError, match="CUDA"):
        rms_norm_backward(x, x, torch.ones(64), torch.ones(4))


def test_entry_points_reject_bad_arguments_without_gpu():
    lib = _lib.lib()

    def forward(rows=4, dim=64, xt=2, wt=2, qt=3, mode=1, pow2=0, x=16, y=16):
        return lib.pcb_rms_norm_fwd(x, xt, rows, dim, 64, None, 0, 16, wt, EPS, None, 0, y, 64, 16, qt, 64, 16, 1, 1,
                                    mode, pow2, 1e-12, 16, None)

    for kwargs in ({"rows": -1}, {"dim": 0}, {"xt": 3}, {"wt": 4}, {"qt": 2}, {"mode": 3}, {"x": None},
                   {"mode": 0, "y": None}):
        assert forward(**kwargs) == _lib.PCB_ERR_INVALID, kwargs
    assert forward(mode=2, pow2=1) == _lib.PCB_ERR_UNSUPPORTED
    assert forward(dim=1 << 30) == _lib.PCB_ERR_UNSUPPORTED
    assert forward(rows=0) == _lib.PCB_OK
    # the backward's workspace has to be there
    assert lib.pcb_rms_norm_bwd(16, 64, 16, 64, 2, 4, 64, None, 0, 16, 2, 16, 16, 64, 16, None, 0,
                                None) == _lib.PCB_ERR_INVALID


@gpu
@pytest.mark.parametrize("dim", [64, 512, 515, 4096, 4101, 16392, 20001])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_row_scales_of_zero_rows_and_non_finite_values(dim, dtype):
    """A row's scale is that of its largest value: not a number where one of them is not."""
    for residual in (False, True):
        x, r, w = _inputs(7, dim, dtype, seed=3, residual=residual)
        x[1] = 0
        if residual:
            r[1] = 0
        x[2, 5], x[3, dim - 1], x[4, 0] = float("inf"), float("nan"), -float("inf")
        for keep in (False, True):
            res = rms_norm_quant(x, w, r, eps=EPS, quant="row", return_y=keep)
            q, scale = res.quant.tensor.float(), res.quant.dequant_scale
            assert int(q[1].count_nonzero()) == 0
            _close(scale[1:2], torch.full((1,), 1e-12 / 448.0, device="cuda").double(), RTOL32, 0.0, "zero row scale")
            for row in (2, 3, 4):  # an infinity's quotient is not a number
                assert bool(torch.isnan(scale[row])) and bool(torch.isnan(q[row]).all())
            assert not keep or bool(torch.isnan(res.y[3]).all())
        good = [0, 5, 6]
        _check_forward(x[good], None if r is None else r[good], w, "row", E4M3, what="rows beside them")


@gpu
@pytest.mark.parametrize("fp8", [E4M3, E5M2])
def test_row_scales_feed_the_per_channel_product(fp8):
    """The norm's QuantResult is one operand of the per-channel BMM as it is, but for the batch."""
    from practice_cuda_b200.registry import QuantResult, get_bmm, get_quant
    from tests._util import assert_bmm_close

    x, r, w = _inputs(300, 512, BF16, seed=31)
    res = rms_norm_quant(x, w, r, eps=EPS, quant="row", fp8_dtype=fp8, return_y=True)
    a = QuantResult(res.quant.tensor[None], res.quant.dequant_scale[None], res.quant.impl, res.quant.granularity,
                    res.quant.meta)
    b = get_quant("b200_per_channel").fn(synthetic((1, 512, 384), std=0.05, seed=32).cuda(), channel_axis=-1, fp8_dtype=fp8)
    out = get_bmm("b200_per_channel_a_k_b_n").fn(a, b)
    expected = (res.quant.tensor.double() * res.quant.dequant_scale.double()[:, None]) @ (
        b.tensor[0].double() * b.dequant_scale[0].double())
    assert_bmm_close(out[0], expected, "norm into product")


@gpu
@pytest.mark.parametrize("rows,dim", [(300, 4096), (40, 515), (70, 8200)])
def test_graph_of_both_passes_on_other_data(rows, dim):
    x, r, w = _inputs(rows, dim, BF16, seed=33)
    for t in (x, r, w):
        t.requires_grad_()
    dy, dh = torch.randn_like(x), torch.randn_like(x)

    def step():
        y, h, quant = rms_norm(x, w, r, quant="block")
        return (y.detach(), h.detach(), quant.tensor.view(torch.uint8), quant.dequant_scale,
                *torch.autograd.grad((y, h), (x, r, w), (dy, dh)))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    other = _inputs(rows, dim, BF16, seed=34)
    with torch.no_grad():
        for t, o in zip((x, r, w), other):
            t.copy_(o)
    dy.copy_(torch.randn_like(dy)), dh.copy_(torch.randn_like(dh))
    graph.replay()
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)
