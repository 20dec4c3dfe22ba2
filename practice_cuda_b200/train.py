"""Training steps of the FP8 decoder (``llama.py``): forward, loss, backward,
gradient clipping and AdamW on synthetic tokens.

``python -m practice_cuda_b200.train [--layers 8 --steps 5 --clip 1.0]``
``torchrun --nproc-per-node N -m practice_cuda_b200.train`` shards the model
with FSDP2 and its FP8 all-gather (one process per GPU).

``--plain`` runs the norms, the loss and the clipping in torch instead of on
this package's kernels (``rms_norm``, ``cross_entropy``, ``grad_clip``).
"""

from __future__ import annotations

import argparse
import os

import torch
import torch.distributed as dist

from .grad_clip import clip_grad_norm_
from .llama import Llama, LlamaConfig


def train_step(model, opt, tokens, *, max_norm: float, plain: bool = False):
    """One step on ``tokens`` [batch, seq + 1]: (loss, gradient norm before clipping)."""
    loss = model(tokens[:, :-1], tokens[:, 1:].contiguous())
    loss.backward()
    if plain:
        norm = torch.nn.utils.clip_grad_norm_(model.parameters(), max_norm)
    else:
        norm = clip_grad_norm_(model.parameters(), max_norm)
    opt.step()
    opt.zero_grad(set_to_none=True)
    return loss.detach(), norm


def build_model(cfg: LlamaConfig, device: torch.device, sharded: bool) -> Llama:
    with torch.device(device):
        model = Llama(cfg)
    model.init_weights(seed=0)
    if not sharded:
        return model.to(torch.bfloat16)
    from torch.distributed.fsdp import MixedPrecisionPolicy, fully_shard

    from .fsdp_fp8 import enable_fp8_all_gather

    enable_fp8_all_gather(model)
    policy = MixedPrecisionPolicy(param_dtype=torch.bfloat16, reduce_dtype=torch.float32)
    for layer in model.layers:
        fully_shard(layer, mp_policy=policy)
    fully_shard(model, mp_policy=policy)
    return model


def main() -> None:
    defaults = LlamaConfig()
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=defaults.n_layers)
    ap.add_argument("--dim", type=int, default=defaults.dim)
    ap.add_argument("--heads", type=int, default=defaults.n_heads)
    ap.add_argument("--ffn", type=int, default=defaults.ffn_dim)
    ap.add_argument("--vocab", type=int, default=defaults.vocab)
    ap.add_argument("--seq", type=int, default=defaults.seq_len)
    ap.add_argument("--scaling", choices=("fp32", "e8m0"), default=defaults.linear_scaling)
    ap.add_argument("--steps", type=int, default=5)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--clip", type=float, default=1.0)
    ap.add_argument("--lr", type=float, default=1e-4)
    ap.add_argument("--plain", action="store_true")
    args = ap.parse_args()

    rank, world = int(os.environ.get("RANK", 0)), int(os.environ.get("WORLD_SIZE", 1))
    device = torch.device("cuda", int(os.environ.get("LOCAL_RANK", 0)))
    torch.cuda.set_device(device)
    if world > 1:
        dist.init_process_group("nccl", device_id=device)
    cfg = LlamaConfig(n_layers=args.layers, dim=args.dim, n_heads=args.heads, ffn_dim=args.ffn, vocab=args.vocab,
                      seq_len=args.seq, linear_scaling=args.scaling, fused=not args.plain)
    model = build_model(cfg, device, world > 1)
    opt = torch.optim.AdamW(model.parameters(), lr=args.lr, fused=True)
    g = torch.Generator().manual_seed(1234 + rank)
    tokens = torch.randint(0, cfg.vocab, (1, cfg.seq_len + 1), generator=g).to(device)

    def step():
        result = train_step(model, opt, tokens, max_norm=args.clip, plain=args.plain)
        if world > 1:
            from .fsdp_fp8 import precompute_fp8_block_weights

            precompute_fp8_block_weights(model)  # quantize each shard once per step
        return result

    for _ in range(args.warmup):
        step()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize(device)
    start.record()
    for _ in range(args.steps):
        loss, norm = step()
    end.record()
    torch.cuda.synchronize(device)
    if rank == 0:
        norm = norm.full_tensor() if hasattr(norm, "full_tensor") else norm
        print(f"loss {loss.item():.4f}  gradient norm {norm.item():.4f}  {start.elapsed_time(end) / args.steps:.2f} ms/step  "
              f"peak memory {torch.cuda.max_memory_allocated(device) / 2 ** 30:.2f} GiB")
    if world > 1:
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
