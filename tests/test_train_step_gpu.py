"""The norm, the loss and the clipping together in a training step of the FP8
decoder.

The fused model and the one with those parts in torch are both measured against
the same weights in fp32 without FP8.  Both quantize the same linears; the fused
one rounds a norm's output once where the other rounds it twice (bf16, then
FP8) and keeps the logits and their gradient in fp32.  So its distance from the
fp32 model may be no larger, but for the chance of which values fall on which
side of a tie: a quarter more is allowed."""

import pytest
import torch

from practice_cuda_b200 import _lib
from practice_cuda_b200.fp8_linear import FP8BlockLinear
from practice_cuda_b200.impls.b200_per_block import b200_per_block_quant
from practice_cuda_b200.llama import Llama, LlamaConfig
from practice_cuda_b200.train import build_model, train_step

pytestmark = pytest.mark.gpu


def _config(scaling, fused):
    return LlamaConfig(n_layers=2, dim=256, n_heads=2, ffn_dim=512, vocab=1000, seq_len=192, linear_scaling=scaling,
                       fused=fused)


def _tokens():
    return torch.randint(0, 1000, (2, 193), generator=torch.Generator().manual_seed(5)).cuda()


def _measured(model, tokens):
    loss = model(tokens[:, :-1], tokens[:, 1:].contiguous())
    loss.backward()
    return loss.item(), {n: p.grad.double() for n, p in model.named_parameters()}


def _in_fp32(cfg):
    model = build_model(cfg, torch.device("cuda"), False).float()
    for module in list(model.modules()):
        for name, child in list(module.named_children()):
            if isinstance(child, FP8BlockLinear):
                linear = torch.nn.Linear(child.in_features, child.out_features, bias=False, device="cuda")
                linear.weight = child.weight
                setattr(module, name, linear)
    return model


@pytest.mark.parametrize("scaling", ["fp32", "e8m0"])
def test_fused_model_is_as_near_the_fp32_one_as_the_plain_one(scaling):
    tokens = _tokens()
    loss64, grads64 = _measured(_in_fp32(_config(scaling, False)), tokens)
    off = []
    for fused in (False, True):
        loss, grads = _measured(build_model(_config(scaling, fused), torch.device("cuda"), False), tokens)
        assert abs(loss - loss64) <= 1e-2 * loss64
        assert grads.keys() == grads64.keys()
        off.append({n: ((g - grads64[n]).norm() / grads64[n].norm()).item() for n, g in grads.items()})
    for name, plain in off[0].items():
        assert off[1][name] <= 1.25 * plain, f"{name}: {off[1][name]:.4f} from the fp32 gradient, in torch {plain:.4f}"
    assert _lib.device_error()[0] == 0


def test_steps_lower_the_loss_and_clip():
    model = build_model(_config("e8m0", True), torch.device("cuda"), False)
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3, fused=True)
    tokens = _tokens()
    losses = []
    for _ in range(12):
        loss, norm = train_step(model, opt, tokens, max_norm=0.5)
        losses.append(loss.item())
        assert torch.isfinite(norm) and norm > 0
    assert losses[-1] < losses[0] - 0.5
    assert _lib.device_error()[0] == 0


def test_linear_with_a_quantized_input():
    lin = FP8BlockLinear(256, 384, bias=False, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(100, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    q = b200_per_block_quant(x.detach(), block_m=1, block_n=128)
    y0, y1 = lin(x), lin(x, q)
    assert torch.equal(y0, y1)
    g = torch.randn_like(y0)
    for a, b in zip(torch.autograd.grad(y0, (x, lin.weight), g), torch.autograd.grad(y1, (x, lin.weight), g)):
        assert torch.equal(a, b)
    for bad in (b200_per_block_quant(x.detach()[:50], block_m=1, block_n=128),
                b200_per_block_quant(x.detach(), block_m=1, block_n=64),
                b200_per_block_quant(x.detach(), block_m=1, block_n=128, fp8_dtype=torch.float8_e5m2)):
        with pytest.raises(ValueError):
            lin(x, bad)
    lin.scaling = "e8m0"  # whose GEMM reads the exponents of the scales alone
    with pytest.raises(ValueError, match="power-of-two"):
        lin(x, q)
    q2 = b200_per_block_quant(x.detach(), block_m=1, block_n=128, pow2_scales=True)
    assert torch.equal(lin(x, q2), lin(x))


def test_no_layers():
    cfg = _config("fp32", True)
    cfg.n_layers = 0
    model = Llama(cfg).cuda().bfloat16()
    model.init_weights()
    tokens = _tokens()
    loss = model(tokens[:, :-1], tokens[:, 1:].contiguous())
    loss.backward()
    assert torch.isfinite(loss) and all(torch.isfinite(p.grad).all() for p in model.parameters())


def test_sharded_gradients_are_clipped(tmp_path):
    """FSDP2 on one rank: the DTensor gradients' norm and their clipped shards."""
    import torch.distributed as dist

    from practice_cuda_b200.grad_clip import clip_grad_norm_

    dist.init_process_group("nccl", init_method=f"file://{tmp_path}/store", rank=0, world_size=1,
                            device_id=torch.device("cuda", 0))
    try:
        model = build_model(_config("e8m0", True), torch.device("cuda", 0), True)
        tokens = _tokens()
        model(tokens[:, :-1], tokens[:, 1:].contiguous()).backward()
        before = [p.grad.full_tensor().double() for p in model.parameters()]
        norm64 = sum(g.square().sum() for g in before).sqrt().item()
        norm = clip_grad_norm_(model.parameters(), 0.25 * norm64)
        assert abs(norm.item() - norm64) <= 2e-6 * norm64
        for p, g in zip(model.parameters(), before):
            expected = 0.25 * norm64 / (norm64 + 1e-6) * g
            assert (p.grad.full_tensor().double() - expected).abs().max() <= 1e-6 * expected.abs().max()
        with pytest.raises(ValueError):
            plain = torch.nn.Parameter(torch.ones(4, device="cuda"))
            plain.grad = torch.ones(4, device="cuda")
            clip_grad_norm_([*model.parameters(), plain], 1.0)
    finally:
        dist.destroy_process_group()
