"""The output projection's cross entropy against plain 64-bit arithmetic.

Tolerances.  A logit is a fp32 tensor-core sum of `dim` exact products, added
16 at a time; each addition is off by at most 2^-23 of the running sum, itself
at most |x| |w|: LOGIT = (dim / 16 + 8) 2^-23 |x| |w|.  A loss is the
difference of two such values plus a few fp32 roundings (RTOL32 of the
logits' size).  G is rounded once to the inputs' type (UNIT) after an
exponential that is off by 2 LOGIT + RTOL32; the products of G with weight and x
add (terms / 16 + 8) 2^-23 of the magnitudes summed, and the gradient is
rounded once more."""

import math

import pytest
import torch

from practice_cuda_b200 import _lib
from practice_cuda_b200.cross_entropy import linear_cross_entropy
from tests._util import synthetic

gpu = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
UNIT = {t: torch.finfo(t).eps / 2 for t in (BF16, F16)}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25}
RTOL32 = 1e-5
IGNORE = -100


def _inputs(tokens, vocab, dim, dtype, seed=0, ignored=0.0, scale=1.0):
    x = synthetic((tokens, dim), std=scale, seed=seed, dtype=dtype).cuda()
    w = synthetic((vocab, dim), std=1.0 / math.sqrt(dim), seed=seed + 1, dtype=dtype).cuda()
    g = torch.Generator().manual_seed(seed + 2)
    target = torch.randint(0, vocab, (tokens,), generator=g)
    target[torch.rand(tokens, generator=g) < ignored] = IGNORE
    return x, w, target.cuda()


def _reference(x, w, target, reduction, dloss):
    """loss, dx, dw in 64 bits, and how far each may be off."""
    tokens, dim = x.shape
    vocab = w.shape[0]
    unit, tiny = UNIT[x.dtype], TINY[x.dtype]
    x64, w64 = x.double(), w.double()
    valid = target != IGNORE
    logits = x64 @ w64.t()
    lse = torch.logsumexp(logits, 1)
    at = torch.where(valid, target, 0)
    nll = torch.where(valid, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    add = 2.0 ** -23
    logit = (dim / 16 + 8) * add * x64.norm(dim=1) * w64.norm(dim=1).max()
    nll_off = torch.where(valid, 2 * logit + RTOL32 * (1 + lse.abs() + logits.abs().amax(1)), 0.0)
    count = valid.sum()
    share = torch.where(valid, dloss.double() / (count if reduction == "mean" else 1), 0.0)
    if reduction == "none":
        loss, loss_off = nll, nll_off
    else:
        div = count if reduction == "mean" else 1
        loss, loss_off = nll.sum() / div, nll_off.sum() / div
    p = torch.exp(logits - lse[:, None])
    onehot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    g = (p - onehot) * share[:, None]
    g_off = (p * (2 * logit + RTOL32)[:, None] + unit * (p - onehot).abs()) * share.abs()[:, None]
    dx, dw = g @ w64, g.t() @ x64
    dx_off = g_off @ w64.abs() + ((vocab / 16 + 8) * add) * (g.abs() @ w64.abs())
    dw_off = g_off.t() @ x64.abs() + ((tokens / 16 + 8) * add) * (g.abs().t() @ x64.abs())
    return (loss, loss_off), (dx, unit * dx.abs() + 1.01 * dx_off + tiny), (dw, unit * dw.abs() + 1.01 * dw_off + tiny)


def _within(actual, expected, off, what):
    assert actual.shape == expected.shape, f"{what}: {tuple(actual.shape)} for {tuple(expected.shape)}"
    d = (actual.double() - expected).abs()
    assert bool((d <= off).all()), f"{what}: off by {d.max().item():.3e}, worst ratio {(d / off).max().item():.2f}"


def _check(x, w, target, reduction="mean", piece=None, dloss=None, what=""):
    if dloss is None:
        dloss = torch.rand(target.shape, generator=torch.Generator().manual_seed(1)).cuda() + 0.5
        dloss = dloss if reduction == "none" else torch.tensor(1.0 if x.dtype == BF16 else 64.0, device="cuda")
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(x, w, target, reduction=reduction, vocab_piece=piece)
    assert loss.dtype == torch.float32
    dx, dw = torch.autograd.grad(loss, (x, w), dloss)
    expected = _reference(x.detach(), w.detach(), target, reduction, dloss)
    for got, (value, off), name in zip((loss, dx, dw), expected, ("loss", "dx", "dw")):
        _within(got.detach(), value, off, f"{what} {name}")
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    assert _lib.device_error()[0] == 0
    return loss.detach(), dx, dw


SHAPES = [
    (1, 1, 8), (1, 2, 16), (3, 127, 64), (2, 128, 72), (7, 129, 136), (128, 256, 64), (129, 257, 128), (256, 512, 256),
    (300, 1000, 200), (257, 4099, 520), (1000, 777, 1024), (1, 40000, 256), (33, 20011, 512), (600, 300, 8),
    (5, 300, 1), (6, 301, 7), (130, 259, 65), (40, 1001, 333),  # widths that are not multiples of 16 bytes
    (800, 515, 72), (900, 300, 77),  # many tokens on rows that do not start on lines
    (300, 600, 768), (300, 600, 776), (140, 1500, 1288),  # tiles of one half, and a ragged second one
]


@gpu
@pytest.mark.parametrize("tokens,vocab,dim", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_shapes(tokens, vocab, dim, dtype):
    x, w, target = _inputs(tokens, vocab, dim, dtype, seed=tokens + vocab + dim)
    _check(x, w, target, "mean", what="mean")
    _check(x, w, target, "none", what="none")
    _check(x, w, target, "sum", what="sum")


@gpu
@pytest.mark.parametrize("tokens,vocab,dim", [(300, 1000, 200), (64, 2500, 128), (520, 4099, 264), (31, 777, 77)])
@pytest.mark.parametrize("piece", [1, 256, 700, 1024, 10 ** 9])
def test_pieces_of_the_vocabulary(tokens, vocab, dim, piece):
    x, w, target = _inputs(tokens, vocab, dim, BF16, seed=piece % 97, ignored=0.2)
    _check(x, w, target, "mean", piece=piece)
    _check(x, w, target, "none", piece=piece)


@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_ignored_tokens(reduction, dtype):
    x, w, target = _inputs(400, 900, 192, dtype, seed=5, ignored=0.4)
    loss, dx, _ = _check(x, w, target, reduction)
    left_out = target == IGNORE
    assert int(dx[left_out].count_nonzero()) == 0
    if reduction == "none":
        assert int(loss[left_out].count_nonzero()) == 0
    # What stands in the rows that are left out does not reach the others.
    other = x.clone()
    other[left_out] *= 1000.0
    loss2, dx2, _ = _check(other, w, target, reduction, what="large rows left out")
    assert torch.equal(loss, loss2) and torch.equal(dx, dx2)


@gpu
def test_every_token_ignored():
    x, w, target = _inputs(70, 300, 64, BF16, seed=6)
    target.fill_(IGNORE)
    x.requires_grad_(), w.requires_grad_()
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(x, w, target, reduction=reduction)
        reference = torch.nn.functional.cross_entropy((x.float() @ w.float().t()).detach(), target, reduction=reduction)
        assert torch.equal(loss.detach(), reference) or (math.isnan(loss.item()) and math.isnan(reference.item()))
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert int(dx.count_nonzero()) == 0 and int(dw.count_nonzero()) == 0


@gpu
def test_sure_and_hopeless_tokens():
    x, w, target = _inputs(256, 512, 128, BF16, seed=7)
    lean = w[target].float() * torch.linspace(-60, 60, 256, device="cuda")[:, None]
    loss, _, _ = _check((x.float() + lean).bfloat16(), w, target, "none")
    assert loss.max().item() > 30 and loss.min().item() < 1e-6 and loss.min().item() >= 0


@gpu
def test_large_and_non_finite_logits():
    x, w, target = _inputs(200, 600, 64, BF16, seed=8, scale=200.0)  # logits of several hundreds
    _check(x, w, target, "mean")
    x, w, target = _inputs(200, 600, 64, BF16, seed=9)
    clean = linear_cross_entropy(x, w, target, reduction="none")
    x[3, 5], x[150, 1] = float("nan"), float("inf")
    loss = linear_cross_entropy(x, w, target, reduction="none")
    bad = torch.zeros(200, dtype=torch.bool, device="cuda")
    bad[3] = bad[150] = True
    assert bool(torch.isnan(loss[bad]).all()) and torch.equal(loss[~bad], clean[~bad])
    assert math.isnan(linear_cross_entropy(x, w, target).item())


@gpu
@pytest.mark.parametrize("spread", [1e-12, 1.0, 1e6])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_weights_of_the_losses(spread, dtype):
    x, w, target = _inputs(150, 700, 96, dtype, seed=10, ignored=0.1)
    dloss = synthetic((150,), seed=11, dtype=torch.float32).cuda() * (spread if dtype == BF16 else min(spread, 1e3))
    dloss[7] = 0.0
    _check(x, w, target, "none", dloss=dloss)
    _check(x, w, target, "none", dloss=torch.zeros_like(dloss))


@gpu
def test_layouts_and_shapes_of_the_arguments():
    x, w, target = _inputs(24, 300, 128, BF16, seed=12)
    plain = _check(x, w, target, "none")
    wide = torch.zeros(24, 200, device="cuda", dtype=BF16)
    for start in (0, 8, 3):  # rows of a wider tensor, 16-byte aligned or not
        view = wide[:, start : start + 128]
        view.copy_(x)
        for a, b in zip(_check(view, w, target, "none"), plain):
            assert torch.equal(a, b)
    wt = w.t().contiguous().t()  # columns contiguous
    for a, b in zip(_check(x, wt, target, "none"), plain):
        assert torch.equal(a, b)
    x3, t2 = x.view(2, 12, 128).requires_grad_(), target.view(2, 12).int()
    loss = linear_cross_entropy(x3, w, t2, reduction="none")
    assert loss.shape == (2, 12) and torch.equal(loss.detach().view(24), plain[0])
    assert torch.autograd.grad(loss.sum(), x3)[0].shape == x3.shape
    same = x[:1].expand(24, 128)  # one row for every token
    _check(same, w, target, "mean", what="expanded")


@gpu
def test_only_the_gradients_that_are_needed():
    x, w, target = _inputs(140, 900, 128, BF16, seed=13)
    _, dx, dw = _check(x, w, target)
    x.requires_grad_()
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, w, target), x)[0], dx)
    x.requires_grad_(False), w.requires_grad_()
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, w, target), w)[0], dw)
    with torch.no_grad():
        assert not linear_cross_entropy(x, w, target).requires_grad


@gpu
def test_differentiable_once():
    x, w, target = _inputs(16, 64, 32, BF16, seed=17)
    x.requires_grad_()
    dx, = torch.autograd.grad(linear_cross_entropy(x, w, target), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@gpu
def test_no_tokens():
    w = torch.ones(10, 16, device="cuda", dtype=BF16, requires_grad=True)
    x = torch.empty(0, 16, device="cuda", dtype=BF16, requires_grad=True)
    target = torch.empty(0, device="cuda", dtype=torch.int64)
    assert math.isnan(linear_cross_entropy(x, w, target).item())
    loss = linear_cross_entropy(x, w, target, reduction="sum")
    assert loss.item() == 0.0
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert dx.shape == (0, 16) and int(dw.count_nonzero()) == 0
    assert linear_cross_entropy(x, w, target, reduction="none").shape == (0,)


@gpu
def test_target_outside_the_vocabulary_is_reported():
    x, w, target = _inputs(100, 300, 64, BF16, seed=14)
    assert _lib.device_error()[0] == 0
    for bad in (300, -1, 1 << 40, -(1 << 40)):
        t = target.clone()
        t[9] = bad
        loss = linear_cross_entropy(x, w, t, reduction="none")
        assert math.isnan(loss[9].item()) and int(torch.isnan(loss).sum()) == 1
        code, site, _ = _lib.device_error()
        assert code == _lib.PCB_ERR_INVALID and site == 19
        xg = x.clone().requires_grad_()
        dx = torch.autograd.grad(linear_cross_entropy(xg, w, t), xg)[0]
        assert bool(torch.isnan(dx[9]).all()) and int(torch.isnan(dx).any(1).sum()) == 1
        assert _lib.device_error()[0] == _lib.PCB_ERR_INVALID and _lib.device_error()[0] == 0


@gpu
def test_gradient_against_differences():
    """Central differences along directions of +-1/16 steps.

    x holds multiples of 1/8 below 4 and w multiples of 1/64 below 1/2, so
    both steps are exact in fp16.  A step moves a logit by about
    sqrt(dim) / 16 * |w| = 0.1: the cubic term is below 2e-3 of the slope's
    terms, G and the gradients are rounded to 2^-11, and the two losses'
    roundings (1e-5 of their size) are divided by the step's 1/8."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randint(-16, 16, (6, 64), generator=g) / 8).to(F16).cuda().requires_grad_()
    w = (torch.randint(-16, 16, (50, 64), generator=g) / 64).to(F16).cuda().requires_grad_()
    target = torch.randint(0, 50, (6,), generator=g).cuda()
    dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, target, reduction="sum"), (x, w))
    for k, (t, grad, step) in enumerate(((x, dx, 1 / 16), (w, dw, 1 / 256))):
        for _ in range(4):
            v = (torch.randint(0, 2, tuple(t.shape), generator=g).cuda() * 2 - 1).to(F16)
            ends = []
            for sign in (1, -1):
                moved = t.detach() + sign * step * v
                assert torch.equal((moved - t.detach()).double(), sign * step * v.double())
                args = (moved, w) if k == 0 else (x, moved)
                ends.append(linear_cross_entropy(*(a.detach() for a in args), target, reduction="none").double().sum())
            slope = (ends[0] - ends[1]) / (2 * step)
            inner = (grad.double() * v.double()).sum()
            terms = grad.double().norm() * math.sqrt(grad.numel())
            assert abs(inner - slope).item() <= 4e-3 * terms.item() + 1e-5 * ends[0].abs().item() / (2 * step)


@gpu
def test_repeatability_stream_and_graph():
    x, w, target = _inputs(500, 3000, 256, BF16, seed=15)
    first = _check(x, w, target, "mean")
    for _ in range(3):
        for a, b in zip(_check(x, w, target, "mean"), first):
            assert torch.equal(a, b)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    with torch.cuda.stream(stream):
        loss = linear_cross_entropy(xg, wg, target)
        grads = torch.autograd.grad(loss, (xg, wg))
    stream.synchronize()
    for a, b in zip((loss, *grads), first):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = linear_cross_entropy(x, w, target)
    x.copy_(x.flip(0))
    target.copy_(target.flip(0))
    graph.replay()
    assert abs(captured.item() - first[0].item()) <= 1e-6 * first[0].item()


@gpu
def test_refusals():
    x, w, target = _inputs(8, 32, 16, BF16, seed=16)
    for bad in (
        lambda: linear_cross_entropy(x.float(), w.float(), target),
        lambda: linear_cross_entropy(x, w.half(), target),
        lambda: linear_cross_entropy(x, w[:, :8], target),
        lambda: linear_cross_entropy(x, w[:0], target),
        lambda: linear_cross_entropy(x, w, target[:4]),
        lambda: linear_cross_entropy(x, w, target.float()),
        lambda: linear_cross_entropy(x, w, target.cpu()),
        lambda: linear_cross_entropy(x, w, target, reduction="batch"),
        lambda: linear_cross_entropy(x, w, target, vocab_piece=0),
    ):
        with pytest.raises(ValueError):
            bad()


def test_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        linear_cross_entropy(torch.ones(2, 8).bfloat16(), torch.ones(4, 8).bfloat16(), torch.zeros(2, dtype=torch.int64))


def test_entry_points_reject_bad_arguments_without_gpu():
    lib = _lib.lib()

    def forward(dtype=2, tokens=4, vocab=8, dim=16, sx=16, reduction=2, x=256, ws=256, nbytes=1 << 30):
        return lib.pcb_linear_ce_fwd(x, sx, 256, 16, dtype, tokens, vocab, dim, 256, IGNORE, reduction, 256, 256, 256,
                                     ws, nbytes, None)

    for kwargs in ({"dtype": 0}, {"dtype": 3}, {"tokens": -1}, {"vocab": 0}, {"dim": 0}, {"reduction": 3}, {"x": None},
                   {"ws": None}, {"ws": 16}, {"nbytes": 8}):
        assert forward(**kwargs) == _lib.PCB_ERR_INVALID, kwargs
    assert forward(tokens=0) == _lib.PCB_OK
    assert forward(sx=17) == _lib.PCB_ERR_LAYOUT and forward(x=264) == _lib.PCB_ERR_LAYOUT
    assert forward(vocab=1 << 40) == _lib.PCB_ERR_UNSUPPORTED
    need = lib.pcb_linear_ce_bwd_workspace_bytes(4096, 32000, 4096, 0, 1, 1)
    # one piece of G (at most 128 MiB) and dX's accumulators, not the logits of the whole vocabulary
    assert need < (128 << 20) + 4096 * 4096 * 4 + (1 << 20)


def test_packed_state_is_checked_without_gpu():
    lib = _lib.lib()
    assert lib.pcb_linear_ce_packed_bytes(0, 32000, 4096) == 0
    assert lib.pcb_linear_ce_packed_bytes(511, 1 << 20, 4096) == 0  # too few tokens
    assert lib.pcb_linear_ce_packed_bytes(4096, 1000, 1024) == 0  # too small a product
    need = lib.pcb_linear_ce_packed_bytes(4096, 32000, 4096)
    assert 4096 * (4096 * 2 + 12) <= need <= 4096 * (4096 * 2 + 12) + 4 * 256

    def forward(tokens, packed, nbytes):
        return lib.pcb_linear_ce_packed_fwd(256, 4096, 256, 4096, 2, tokens, 32000, 4096, 256, IGNORE, 2, 256, 256, 256,
                                            packed, nbytes, 256, 1 << 40, None)

    def backward(tokens, packed, nbytes):
        return lib.pcb_linear_ce_packed_bwd(256, 4096, 256, 4096, 2, tokens, 32000, 4096, 256, IGNORE, 2, 256, 256,
                                            packed, nbytes, 256, 256, 4096, None, 4096, 0, 256, 1 << 40, None)

    for call in (forward, backward):
        assert call(4096, None, need) == _lib.PCB_ERR_INVALID
        assert call(4096, 128, need) == _lib.PCB_ERR_INVALID
        assert call(4096, 256, need - 1) == _lib.PCB_ERR_INVALID
        assert call(8, 256, need) == _lib.PCB_ERR_INVALID  # state that nothing would write
        assert call(0, None, 0) == _lib.PCB_OK


def _mask(name, tokens):
    """Tokens that are left out."""
    out = torch.zeros(tokens, dtype=torch.bool)
    if name == "first":
        out[0] = True
    elif name == "last":
        out[-1] = True
    elif name == "scattered":
        out = torch.rand(tokens, generator=torch.Generator().manual_seed(17)) < 0.4
    elif name == "one tile left":
        out[256:] = True
    elif name == "one more than a tile left":
        out[:tokens - 257] = True
    elif name == "one left":
        out[:] = True
        out[tokens // 2] = False
    elif name == "all":
        out[:] = True
    return out.cuda()


@gpu
@pytest.mark.parametrize("tokens,vocab,dim", [(515, 33001, 4104), (2100, 8200, 4032)])
@pytest.mark.parametrize("mask", ["none", "first", "last", "scattered", "one tile left", "one more than a tile left",
                                  "one left"])
def test_tokens_left_out_of_large_products(tokens, vocab, dim, mask):
    x, w, target = _inputs(tokens, vocab, dim, BF16, seed=tokens)
    left_out = _mask(mask, tokens)
    target[left_out] = IGNORE
    assert _lib.lib().pcb_linear_ce_packed_bytes(tokens, vocab, dim) > 0
    for reduction, piece in (("mean", None), ("none", None), ("sum", 2048)):
        loss, dx, dw = _check(x, w, target, reduction, piece=piece, what=reduction)
        assert int(dx[left_out].count_nonzero()) == 0
        if reduction == "none":
            assert int(loss[left_out].count_nonzero()) == 0
    score = linear_cross_entropy(x, w, target, reduction="none")
    assert torch.equal(score, linear_cross_entropy(x.requires_grad_(), w, target, reduction="none").detach())


@gpu
def test_large_product_of_no_token():
    x, w, target = _inputs(600, 30000, 4096, F16, seed=6)
    target.fill_(IGNORE)
    assert _lib.lib().pcb_linear_ce_packed_bytes(600, 30000, 4096) > 0
    x.requires_grad_(), w.requires_grad_()
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(x, w, target, reduction=reduction)
        assert bool(torch.isnan(loss)) if reduction == "mean" else int(loss.count_nonzero()) == 0
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert int(dx.count_nonzero()) == 0 and int(dw.count_nonzero()) == 0


@gpu
def test_gradients_of_large_products_on_rows_of_other_strides():
    """dX whose rows do not suit TMA (a C caller's), one gradient at a time, an output of odd stride."""
    tokens, vocab, dim = 700, 24001, 4104
    x, w, target = _inputs(tokens, vocab, dim, BF16, seed=3, ignored=0.5)
    _, dx, dw = _check(x, w, target, "mean")
    x1, w1 = x.detach().requires_grad_(), w.detach().requires_grad_()
    only_x, = torch.autograd.grad(linear_cross_entropy(x1, w, target), x1)
    only_w, = torch.autograd.grad(linear_cross_entropy(x, w1, target), w1)
    (_, _), (ex, ox), (ew, ow) = _reference(x, w, target, "mean", torch.tensor(1.0, device="cuda"))
    _within(only_x, ex, ox, "dx alone")
    _within(only_w, ew, ow, "dw alone")
    lib, code = _lib.lib(), _lib.PCB_DTYPE[BF16]
    stream = torch.cuda.current_stream().cuda_stream
    packed = torch.empty(lib.pcb_linear_ce_packed_bytes(tokens, vocab, dim), dtype=torch.uint8, device="cuda")
    stats, count = torch.empty(2 * tokens, device="cuda"), torch.empty(1, device="cuda")
    loss, one = torch.empty((), device="cuda"), torch.ones((), device="cuda")
    ws = torch.empty(lib.pcb_linear_ce_fwd_workspace_bytes(tokens, vocab), dtype=torch.uint8, device="cuda")
    args = (x.data_ptr(), dim, w.data_ptr(), dim, code, tokens, vocab, dim, target.data_ptr(), IGNORE, 2)
    forward = lambda nbytes: lib.pcb_linear_ce_packed_fwd(
        *args, loss.data_ptr(), stats.data_ptr(), count.data_ptr(), packed.data_ptr(), nbytes, ws.data_ptr(),
        ws.numel(), stream)
    assert forward(packed.numel() - 1) != 0  # refused before anything runs
    assert forward(packed.numel()) == 0
    for piece in (0, 4096):
        out = torch.full((tokens, dim + 1), 7.0, dtype=BF16, device="cuda")
        ws2 = torch.empty(lib.pcb_linear_ce_bwd_workspace_bytes(tokens, vocab, dim, piece, 1, 0), dtype=torch.uint8,
                          device="cuda")
        assert lib.pcb_linear_ce_packed_bwd(
            *args, stats.data_ptr(), count.data_ptr(), packed.data_ptr(), packed.numel(), one.data_ptr(),
            out.data_ptr(), dim + 1, None, dim, piece, ws2.data_ptr(), ws2.numel(), stream) == 0
        _within(out[:, :dim], ex, ox, f"dx of stride {dim + 1}, piece {piece}")
        assert bool((out[:, dim] == 7.0).all())


@gpu
@pytest.mark.parametrize("tokens,vocab,dim", [(2, 40, 16), (9, 300, 72), (100, 517, 77), (300, 900, 192),
                                              (600, 300, 64), (515, 33001, 4104), (900, 700, 260)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_rows_left_out_reach_nothing(tokens, vocab, dim, reduction, value):
    x, w, target = _inputs(tokens, vocab, dim, BF16, seed=dim, ignored=0.5)
    target[tokens // 2] = IGNORE
    target[0] = 1
    left_out = target == IGNORE
    x[left_out] = 0.0
    expected = _check(x, w, target, reduction, what="zeros")
    x[left_out] = value
    dloss = torch.rand(target.shape, generator=torch.Generator().manual_seed(1)).cuda() + 0.5
    dloss = dloss if reduction == "none" else torch.tensor(1.0, device="cuda")
    x1, w1 = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(x1, w1, target, reduction=reduction)
    got = (loss.detach(), *torch.autograd.grad(loss, (x1, w1), dloss))
    for a, b, name in zip(got, expected, ("loss", "dx", "dw")):
        assert torch.equal(a, b), name
    loss = linear_cross_entropy(x, w1, target, reduction=reduction)
    assert torch.equal(torch.autograd.grad(loss, w1, dloss)[0], expected[2])
    assert _lib.device_error()[0] == 0


@gpu
@pytest.mark.parametrize("tokens,vocab,dim", [(515, 33001, 4104), (300, 900, 192)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_entry_points_without_packed_state(tokens, vocab, dim, reduction):
    """pcb_linear_ce_fwd and _bwd, at a size that the packed passes would pack and at one that they would not:
    what x holds for tokens that are left out reaches nothing."""
    x, w, target = _inputs(tokens, vocab, dim, BF16, seed=dim, ignored=0.4)
    left_out = target == IGNORE
    lib, code = _lib.lib(), _lib.PCB_DTYPE[BF16]
    assert (lib.pcb_linear_ce_packed_bytes(tokens, vocab, dim) > 0) == (tokens > 500)
    stream = torch.cuda.current_stream().cuda_stream
    red = ["none", "sum", "mean"].index(reduction)
    one = torch.rand(tokens if red == 0 else 1, generator=torch.Generator().manual_seed(1)).cuda() + 0.5
    ws = torch.empty(lib.pcb_linear_ce_fwd_workspace_bytes(tokens, vocab), dtype=torch.uint8, device="cuda")
    ws2 = torch.empty(lib.pcb_linear_ce_bwd_workspace_bytes(tokens, vocab, dim, 0, 1, 1), dtype=torch.uint8, device="cuda")

    def run():
        ws.fill_(0xff), ws2.fill_(0xff)  # NaN, whatever they are read as
        args = (x.data_ptr(), dim, w.data_ptr(), dim, code, tokens, vocab, dim, target.data_ptr(), IGNORE, red)
        loss, stats, count = (torch.empty(n, device="cuda") for n in (one.numel(), 2 * tokens, 1))
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        assert lib.pcb_linear_ce_fwd(*args, loss.data_ptr(), stats.data_ptr(), count.data_ptr(), ws.data_ptr(),
                                     ws.numel(), stream) == 0
        assert lib.pcb_linear_ce_bwd(*args, stats.data_ptr(), count.data_ptr(), one.data_ptr(), dx.data_ptr(), dim,
                                     dw.data_ptr(), dim, 0, ws2.data_ptr(), ws2.numel(), stream) == 0
        return loss, dx, dw

    x[left_out] = 0.0
    clean = run()
    expected = _reference(x, w, target, reduction, one if red == 0 else one[0])
    for got, (value, off), name in zip(clean, expected, ("loss", "dx", "dw")):
        _within(got.view(value.shape), value, off, name)
    for value in (float("nan"), float("-inf")):
        x[left_out] = value
        for a, b, name in zip(run(), clean, ("loss", "dx", "dw")):
            assert torch.equal(a, b), f"{name} with {value}"
    assert _lib.device_error()[0] == 0


@gpu
def test_forward_mode_is_refused():
    """No tangent is dropped without a word, whatever else the call needs."""
    import torch.autograd.forward_ad as forward_ad

    x, w, target = _inputs(16, 64, 32, BF16, seed=18)
    tangent = torch.ones_like(x)
    with forward_ad.dual_level():
        dual_x, dual_w = forward_ad.make_dual(x, tangent), forward_ad.make_dual(w, torch.ones_like(w))
        for args in ((dual_x, w), (x, dual_w), (x.clone().requires_grad_(), dual_w),
                     (forward_ad.make_dual(x.view(2, 8, 32), tangent.view(2, 8, 32)), w)):
            with pytest.raises(NotImplementedError, match="jvp"):
                linear_cross_entropy(*args, target.view(args[0].shape[:-1]))
            with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
                linear_cross_entropy(*args, target.view(args[0].shape[:-1]))
        assert not linear_cross_entropy(x, w, target).requires_grad


@gpu
def test_error_of_the_loss_beside_another_kernels():
    """Two kernels report in one interval: both errors are read, one after the other."""
    from practice_cuda_b200.registry import get_bmm, get_quant

    _lib.device_error()  # clear
    a, b = synthetic((1, 128, 128), seed=30).cuda(), synthetic((1, 128, 128), seed=31).cuda()
    quant = get_quant("b200_per_channel").fn
    qa, qb = quant(a, channel_axis=-2), quant(b, channel_axis=-1)
    _lib.check(_lib.lib().pcb_debug_inject_error(_lib.PCB_ERR_TIMEOUT), "inject")
    get_bmm("b200_per_channel_a_k_b_n").fn(qa, qb)
    x, w, target = _inputs(10, 300, 64, BF16, seed=14)
    target[3] = 300
    linear_cross_entropy(x, w, target)
    codes = [_lib.device_error()[:2] for _ in range(3)]
    assert codes == [(_lib.PCB_ERR_TIMEOUT, 4), (_lib.PCB_ERR_INVALID, 19), (0, 0)]


def test_workspace_sizes_of_any_arguments_without_gpu():
    """Sizes whose sums pass 64 bits: no crash, and a piece beyond the vocabulary is the vocabulary."""
    import subprocess
    import sys

    program = """
import ctypes, sys
lib = ctypes.CDLL(sys.argv[1])
i64 = ctypes.c_int64
def sized(name, *args):
    fn = getattr(lib, name)
    fn.restype, fn.argtypes = i64, [i64] * len(args)
    return fn(*args)
big = 2 ** 63 - 1
whole = sized("pcb_linear_ce_bwd_workspace_bytes", 300, 1000, 200, 1024, 1, 1)
assert whole > 0
for piece in (1025, 10 ** 9, 2 ** 31, 2 ** 62, big - 300, big):
    assert sized("pcb_linear_ce_bwd_workspace_bytes", 300, 1000, 200, piece, 1, 1) == whole, piece
    assert sized("pcb_linear_ce_packed_bwd_workspace_bytes", 300, 1000, 200, piece, 1, 1) == whole, piece
for tokens, vocab, dim in ((big, 1000, 200), (300, big, 200), (300, 1000, big), (big, big, big), (300, big - 100, 64),
                           (2 ** 27, 1000, 200), (300, 2 ** 27, 200), (2 ** 26, 2 ** 26, 8)):
    # what the passes refuse needs no room
    assert sized("pcb_linear_ce_bwd_workspace_bytes", tokens, vocab, dim, 0, 1, 1) == 0, (tokens, vocab, dim)
    assert sized("pcb_linear_ce_packed_bwd_workspace_bytes", tokens, vocab, dim, 0, 1, 1) == 0, (tokens, vocab, dim)
    assert sized("pcb_linear_ce_packed_bytes", tokens, vocab, dim) == 0, (tokens, vocab, dim)
for tokens, vocab in ((big, 1000), (300, big), (big, big), (300, big - 100), (2 ** 27, 10), (10, 2 ** 27), (2 ** 26, 2 ** 26)):
    assert sized("pcb_linear_ce_fwd_workspace_bytes", tokens, vocab) == 0, (tokens, vocab)
"""
    done = subprocess.run([sys.executable, "-c", program, _lib.LIB_PATH], capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stderr)


@gpu
def test_a_piece_beyond_the_vocabulary():
    x, w, target = _inputs(40, 300, 64, BF16, seed=19)
    first = _check(x, w, target)
    for piece in (10 ** 6, 2 ** 62, 2 ** 63 - 1):
        for a, b in zip(_check(x, w, target, piece=piece), first):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("tokens", [60, 290])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradients_of_sure_tokens(tokens, dtype):
    """Tokens whose target has all but 1e-6 to 1e-3 of the probability keep what is left of the gradient's digits.

    weight is half an identity and a row of x has its target's column, one other, and
    -400 elsewhere, so a logit is one exact product and a probability of two terms: e in
    1 + e is rounded once, by 2^-24 at most, and dx is 0.5 G, rounded to the type as G
    and as dx; RTOL32 covers e's own exponential and the logarithm."""
    vocab = 256
    w = (0.5 * torch.eye(vocab)).to(dtype).cuda()
    x = torch.full((tokens, vocab), -400.0)
    g = torch.Generator().manual_seed(20)
    target = torch.randint(0, vocab, (tokens,), generator=g)
    other = (target + torch.randint(1, vocab, (tokens,), generator=g)) % vocab
    rows = torch.arange(tokens)
    x[rows, target] = 10.0
    x[rows, other] = 10.0 - torch.randint(56, 112, (tokens,), generator=g) / 4  # e of exp(-7) to exp(-13.9)
    x, target, other, rows = x.to(dtype).cuda().requires_grad_(), target.cuda(), other.cuda(), rows.cuda()
    for reduction in ("sum", "none"):
        loss = linear_cross_entropy(x, w, target, reduction=reduction)
        dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
        logits = 0.5 * x.detach().double()
        e = torch.exp(logits[rows, other] - logits[rows, target])
        if reduction == "none":
            _within(loss.detach(), torch.log1p(e), 2.0 ** -24 + RTOL32 * e, "loss")
        for column, sign in ((target, -1.0), (other, 1.0)):
            expected = sign * 0.5 * e / (1 + e)
            off = 0.5 * 2.0 ** -24 + (2 * UNIT[dtype] * 1.01 + RTOL32) * expected.abs() + TINY[dtype]
            _within(dx[rows, column], expected, off, f"{reduction} {sign:+.0f}")
        rest = dx.clone()
        rest[rows, target] = rest[rows, other] = 0.0
        assert int(rest.count_nonzero()) == 0


@gpu
def test_mean_loss_of_long_products():
    """The tensor cores truncate as they add, which moves every logit towards zero and, since
    the errors agree in sign, a mean loss with them.  Between two promotions (512 products, 32
    additions of 16) each addition loses less than 2^-23 of the running sum, on average half of
    that, of a sum that has on average come half of its way: 32 * 2^-23 / 4 < 1e-6 of a logit.
    The loss is the difference of the target's logit and the expected one."""
    tokens, vocab, dim = 2000, 4000, 4096
    g = torch.Generator(device="cuda").manual_seed(21)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    weight = 0.02 * normal(vocab, dim)
    target = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    lean = torch.rand((tokens, 1), generator=g, device="cuda") * 16.0 / (0.02 ** 2 * dim)
    x, w = (normal(tokens, dim) + lean * weight[target]).bfloat16(), weight.bfloat16()
    logits = x.double() @ w.double().t()
    lse = torch.logsumexp(logits, 1)
    at = logits.gather(1, target[:, None])[:, 0]
    expected = (torch.exp(logits - lse[:, None]) * logits).sum(1)
    loss = linear_cross_entropy(x, w, target).double()
    off = (loss - (lse - at).mean()).abs()
    bound = 1e-6 * (at - expected).abs().mean() + 2.0 ** -23 * (lse - at).mean()
    assert bool(off <= bound), f"mean loss off by {off.item():.3e}, {(off / bound).item():.2f} of the bound"


@gpu
@pytest.mark.parametrize("tokens,vocab,dim,first,second", [
    (60, 700, 136, 0.0, 0.3),  # single CTAs
    (500, 3000, 256, 0.3, 0.0),
    (2100, 8200, 4032, 0.1, 0.7),  # packed: another number of tiles
    (2100, 8200, 4032, 0.5, 0.0),  # packed, then none left out
])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_graph_of_both_passes_on_other_data(tokens, vocab, dim, first, second, reduction):
    x, w, target = _inputs(tokens, vocab, dim, BF16, seed=22, ignored=first)
    x.requires_grad_(), w.requires_grad_()
    dloss = torch.rand(tokens if reduction == "none" else (), device="cuda") + 0.5

    def step():
        loss = linear_cross_entropy(x, w, target, reduction=reduction)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w), dloss))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed, ignored in ((23, second), (24, first)):
        other = _inputs(tokens, vocab, dim, BF16, seed=seed, ignored=ignored)
        with torch.no_grad():
            x.copy_(other[0]), w.copy_(other[1]), target.copy_(other[2])
        dloss.copy_(torch.rand_like(dloss) + 0.5)
        for t in captured:
            t.fill_(float("nan"))
        graph.replay()
        for a, b, name in zip(captured, step(), ("loss", "dx", "dw")):
            assert torch.equal(a, b), name
    assert _lib.device_error()[0] == 0


@gpu
def test_the_weight_is_not_copied():
    """Rows that suit TMA, if not whole lines: a copy of the weight would cost more than it gives, and stay until the
    backward pass."""
    x, w, target = _inputs(1024, 30000, 1032, BF16, seed=25)
    w.requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    loss = linear_cross_entropy(x, w, target)
    weight = w.numel() * w.element_size()
    assert torch.cuda.max_memory_allocated() - before < weight // 2
    dw, = torch.autograd.grad(loss, w)
    assert dw.shape == w.shape


@gpu
@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("dim", [512, 576, 640, 704, 768, 1216, 4096])
def test_logits_are_promoted_every_512_products(tokens, dim):
    """A logit whose first 16 products make 2048 and whose further additions are each 15/16 of its last place: those of
    the same 512 products may be lost, 31 of them, the others not.  The other logit is 2048 itself."""
    x = torch.ones(tokens, dim, device="cuda", dtype=BF16)
    w = torch.zeros(2, dim, device="cuda", dtype=BF16)
    w[:, :16] = 128.0
    place = 2.0 ** -12
    w[0, 16:] = 15 / 256 * place
    target = torch.zeros(tokens, device="cuda", dtype=torch.int64)
    loss = linear_cross_entropy(x, w, target, reduction="none").double()
    ahead = (dim - 16) * 15 / 256 * place  # of the first logit
    # 31 additions that are lost, one rounding a promotion, and the loss's own (a slope of a half at most)
    off = 0.5 * place * (31 * 15 / 16 + 0.5 * math.ceil(dim / 512)) + 2.0 ** -23
    _within(loss, torch.full_like(loss, math.log1p(math.exp(-ahead))), off, "loss")


def test_one_workspace_serves_either_backward_pass_without_gpu():
    lib = _lib.lib()
    for tokens in (1, 100, 515, 4096, 20000):
        for vocab in (300, 8200, 16000, 32000, 50001, 128000):
            for dim in (64, 1000, 4096):
                for piece in (0, 256, 5000, 1 << 40):
                    for want in ((1, 1), (1, 0), (0, 1)):
                        args = (tokens, vocab, dim, piece, *want)
                        packed = lib.pcb_linear_ce_packed_bwd_workspace_bytes(*args)
                        assert 0 < packed <= lib.pcb_linear_ce_bwd_workspace_bytes(*args), args


@gpu
@pytest.mark.parametrize("tokens,vocab,dim,piece,ignored", [
    (1, 700, 2048, None, 0.0), (1, 5000, 771, None, 0.0), (7, 1500, 4096, 512, 0.0), (40, 3000, 1032, None, 0.3),
    (128, 257, 2056, None, 0.0), (129, 9000, 1001, None, 0.0), (300, 4099, 2048, 1024, 0.2), (700, 24001, 4104, None, 0.5),
    (2100, 8200, 4032, None, 0.0), (2100, 8200, 4032, 2048, 0.4),
])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_of_gradients_are_not_moved_as_a_whole(tokens, vocab, dim, piece, ignored, dtype):
    """G holds a token's own entry beyond 16 bits: the entry multiplies all of a row, so its rounding would move the row as
    one, by up to 2^-9 (bf16).

    k is a row's component along the exact one.  Rounding the result's elements moves it by the sum of
    independent errors of at most UNIT, uniform at most (UNIT / sqrt(3) each); so do the roundings of the other
    entries of G, through the part of their rows that lies along this one.  Seven times their root of
    summed squares is allowed, and RTOL32 for the arithmetic between."""
    x, w, target = _inputs(tokens, vocab, dim, dtype, seed=dim, ignored=ignored)
    target[0] = 3
    target[tokens // 2] = 3  # two tokens of one target
    g = torch.Generator().manual_seed(26)
    dloss = (torch.rand(tokens, generator=g) + 0.5).cuda() * (1.0 if dtype == BF16 else 64.0)
    x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(x, w, target, reduction="none", vocab_piece=piece)
    dx, dw = torch.autograd.grad(loss, (x, w), dloss)
    x64, w64 = x.detach().double(), w.detach().double()
    valid = target != IGNORE
    at = torch.where(valid, target, 0)[:, None]
    p = torch.softmax(x64 @ w64.t(), 1) * torch.where(valid, dloss.double(), 0.0)[:, None]
    full = p.scatter_add(1, at, torch.where(valid, -dloss.double(), 0.0)[:, None])
    p.scatter_(1, at, 0.0)  # the entries that are rounded
    unit = UNIT[dtype] / math.sqrt(3.0)

    def along(got, exact, entries, rows):
        """k of each row, and how far it may be off, for exact = (entries and the own ones) @ rows."""
        square = exact.square().sum(1)
        k = (got.double() * exact).sum(1) / square - 1
        rounded = exact.pow(4).sum(1)
        others = (entries.square() * (exact @ rows.t()).square()).sum(1)
        return k.abs(), 7 * unit * torch.sqrt(rounded + others) / square + RTOL32 + 2 * LOGIT

    LOGIT = ((dim / 16 + 8) * 2.0 ** -23 * x64.norm(dim=1).max() * w64.norm(dim=1).max()).item()
    k, off = along(dx, full @ w64, p, w64)
    assert bool((k <= off)[valid].all()), f"dx moved by {k[valid].max().item():.2e}, {(k / off)[valid].max().item():.2f} of its bound"
    rows = torch.unique(target[valid])
    k, off = along(dw[rows], full.t()[rows] @ x64, p.t()[rows], x64)
    assert bool((k <= off).all()), f"dw moved by {k.max().item():.2e}, {(k / off).max().item():.2f} of its bound"


@gpu
@pytest.mark.parametrize("tokens", [5, 70, 1000, 9000])
@pytest.mark.parametrize("pattern", ["one", "two in turn", "blocks", "random", "far apart"])
def test_tokens_that_share_targets(tokens, pattern):
    """Lists of a target's tokens: every length, neighbours, tokens that are thousands apart, ignore_index among the columns."""
    vocab, dim = 301, 72
    x, w, target = _inputs(tokens, vocab, dim, BF16, seed=27)
    i = torch.arange(tokens, device="cuda")
    if pattern == "one":
        target[:] = 300
    elif pattern == "two in turn":
        target = i % 2 * 255
    elif pattern == "blocks":
        target = i // 9 % vocab
    elif pattern == "far apart":
        target = torch.where(i < tokens // 2, i % 150, 200 + i % 90)
        target[0] = target[-1] = 299
    first = _check(x, w, target, "mean", what=pattern)
    for a, b in zip(_check(x, w, target, "mean", what=pattern), first):
        assert torch.equal(a, b)
    # A column may be what marks the tokens that are left out.
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = target == int(target[-1])
    got = torch.autograd.grad(linear_cross_entropy(xg, wg, target, reduction="sum", ignore_index=int(target[-1])), (xg, wg))
    want = torch.autograd.grad(linear_cross_entropy(xg, wg, target.masked_fill(out, IGNORE), reduction="sum"), (xg, wg))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
