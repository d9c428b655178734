"""Analog inference of a transformer with the layer shapes of GPT-2 small: every linear layer of
the blocks runs on mapped analog tiles, everything else stays digital fp32.

    python -m aihwkit_b200.gpt2_inference [--layers 12] [--batch 16] [--seq 1024] [--steps 5]
                                          [--adapters 4 --rank 16 [--adapt-steps 3]]
    python -m torch.distributed.run --nproc-per-node N ... -m aihwkit_b200.gpt2_inference ...

Shapes only: the weights are random (N(0, 0.02), seeded), the token ids uniform over the
vocabulary; no checkpoint and no text is involved.  Per block: QKV 768 -> 2304, attention output
768 -> 768, MLP 768 -> 3072 -> 768.  Each of them is a mapped-tile layer
(``TileModuleArray``, src/aihwkit/simulator/tiles/array.py:30-198) with tiles of at most 512 x 512
(768 -> [384, 384], 2304 -> 4 x 461 + 460, 3072 -> 6 x 512) and the inference IO settings
(8-bit DAC / ADC, out_noise 0.04, additive weight noise 0.0175, ABS_MAX noise management).
Embeddings, LayerNorm, attention, GELU, residuals and the vocabulary projection are fp32 torch ops,
as they are digital in the reference too (``AnalogLinear`` only replaces ``nn.Linear``,
src/aihwkit/nn/conversion.py).

Two ways to use N ranks (``--shard``):
  ``sequences`` (default): sequences are independent, so every rank takes ``batch / N`` sequences
      and holds all tiles; no collective on the data path.
  ``tiles``: the tiles of every analog layer are dealt to the ranks - over the in-splits first,
      over the out-splits where a layer has fewer in-splits than ranks (768 -> 2 in-splits) - every
      rank computes the partial output of its block of tiles for ALL tokens, and one NCCL
      all-reduce per layer adds the partial outputs up (``TileModuleArray``'s ``result.add_`` over
      in-splits, tiles/array.py:173-176, across GPUs).  The digital parts run replicated.
With ``--adapters N`` every analog layer has a pool of N low-rank adapters beside its tiles, the sequences of the
batch use them in turn, and the digital parts of the blocks (residual sums, LayerNorm, dropout in training) run on the
library's own kernels (:mod:`aihwkit_b200.digital`).  ``--adapt-steps K`` then takes K training steps on the adapters and
the norms, in one process: the conductances stay as they were programmed, gradients pass the tiles through their transposed
product.

Prints one JSON line (rank 0): tokens/s of the whole forward, the share of the analog layers, and
their logical TFLOP/s.
"""

from __future__ import annotations

import argparse
import json
import os
from typing import List, Optional

import torch
import torch.nn.functional as F

VOCAB, N_POS = 50257, 1024


def inference_config(seed: int, max_tile: int = 512, adapted: bool = False):
    from .rpu_base import devices as D

    p = D.AnalogTileParameter()
    io = p.forward_io
    io.inp_res = io.out_res = 1.0 / 254.0
    io.out_noise = 0.04
    io.w_noise = 0.0175
    io.w_noise_type = D.WeightNoiseType.AdditiveConstant
    io.out_bound, io.inp_bound = 10.0, 1.0
    io.noise_management = D.NoiseManagementType.AbsMax
    io.bound_management = D.BoundManagementType.None_
    p.update.pulse_type = D.PulseType.None_
    if adapted:
        p.backward_io.is_perfect = True  # gradients of digital adapters are a digital product with the weights
    return p._config(max_tile, max_tile, D.IdealResistiveDeviceParameter(), seed=seed)


class AnalogLinear:
    """``y = sum over tiles of alpha_tile * tile(x) + bias``: every tile stores its block of the
    weight matrix divided by ``alpha_tile = max|w_tile|`` so that it fills the conductance range
    [-1, 1] (the reference's weight-scaling omega = 1, layer-wise per tile,
    src/aihwkit/simulator/tiles/periphery.py:437-500); the scales and the digital bias are applied
    inside the mapped layer's kernels, so a layer is two launches (DAC, MVM)."""

    def __init__(self, in_features: int, out_features: int, device: int, seed: int,
                 gen: torch.Generator, max_tile: int = 512, shard_tiles: bool = False, adapters: int = 0,
                 rank: int = 16):
        from .rpu_base import tiles as T
        from .sharded import ShardedTileArray

        w = torch.randn(out_features, in_features, generator=gen) * 0.02
        cfg = inference_config(seed, max_tile, adapted=True) if adapters else inference_config(seed, max_tile)
        self.sharded = None
        if shard_tiles:
            # this rank's block of the layer's tiles; the ranks' partial outputs are all-reduced
            self.sharded = ShardedTileArray(
                out_features, in_features, max_tile, max_tile,
                lambda b, e, ob, oe: T.TileArray(cfg, out_features, in_features, max_tile, max_tile,
                                                 cuda_device=device, in_split_range=(b, e),
                                                 out_split_range=(ob, oe)),
                two_d=True)
            self.array = self.sharded.local
        else:
            self.array = T.TileArray(cfg, out_features, in_features, max_tile, max_tile,
                                     cuda_device=device)
        self.array.set_seed(seed)
        self.array.set_weights(w, weight_scaling_omega=1.0)
        self.array.set_bias(torch.zeros(out_features))
        self.in_features, self.out_features = in_features, out_features
        self.adapters = None
        if adapters:
            from .digital import LowRankAdapters

            if shard_tiles:
                raise RuntimeError("adapters are built for layers whose tiles are all on one GPU")
            self.adapters = LowRankAdapters(adapters, in_features, out_features, rank, device=f"cuda:{device}",
                                            generator=torch.Generator().manual_seed(seed))

    @property
    def n_tiles(self) -> int:
        return self.array.num_in_splits * self.array.num_out_splits

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        y = self.array.forward(x.reshape(-1, self.in_features), is_test=True, non_blocking=True)
        if self.sharded is not None:
            y = self.sharded.reduce(y, dst=None)  # all-reduce of the shards' partial outputs
        return y.reshape(*x.shape[:-1], self.out_features)

    def adapted(self, x: torch.Tensor, adapter_ids: torch.Tensor, row_starts: torch.Tensor) -> torch.Tensor:
        """The layer with its adapters, differentiable in ``x`` and the adapters."""
        y = _Tiles.apply(x, self.array)
        grad = torch.is_grad_enabled() and any(t.requires_grad for t in (x, y, self.adapters.a, self.adapters.b))
        return self.adapters(y, x, adapter_ids, row_starts, out=None if grad else y)


class _Tiles(torch.autograd.Function):
    """The product of a mapped layer; its gradient is the layer's backward product (the weights take no part)."""

    @staticmethod
    def forward(ctx, x, array):
        ctx.array = array
        return array.forward(x, is_test=True, non_blocking=True)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        return ctx.array.backward(gy, non_blocking=True), None


class Adaptation:
    """One pass of a model with adapters: the adapter of every sequence, and the dropout in front of the residual sums
    (``p``, ``seed``; the dropouts of a pass number their calls from ``call`` on, two to a block)."""

    def __init__(self, adapter_ids: torch.Tensor, seq: int, p: float = 0.0, seed: int = 0, call: int = 0):
        self.adapter_ids = adapter_ids.to(torch.int32)
        self.row_starts = torch.arange(adapter_ids.numel() + 1, dtype=torch.int32, device=adapter_ids.device) * seq
        self.p, self.seed, self.call = p, seed, call

    def linear(self, layer: AnalogLinear):
        return lambda x: layer.adapted(x, self.adapter_ids, self.row_starts)

    def add_norm(self, x, h, norm):
        from . import digital

        y, h = digital.add_layer_norm(x, h, norm[0], norm[1], p=self.p, seed=self.seed, call=self.call)
        self.call = (self.call + 1) & 0xFFFFFFFF
        return y, h


class Block:
    def __init__(self, d_model: int, n_head: int, device: int, seed: int, gen: torch.Generator,
                 shard_tiles: bool = False, adapters: int = 0, rank: int = 16):
        dev = f"cuda:{device}"
        more = dict(shard_tiles=shard_tiles, adapters=adapters, rank=rank)
        self.n_head = n_head
        self.ln1_w, self.ln1_b = torch.ones(d_model, device=dev), torch.zeros(d_model, device=dev)
        self.ln2_w, self.ln2_b = torch.ones(d_model, device=dev), torch.zeros(d_model, device=dev)
        self.qkv = AnalogLinear(d_model, 3 * d_model, device, seed + 1, gen, **more)
        self.proj = AnalogLinear(d_model, d_model, device, seed + 2, gen, **more)
        self.fc = AnalogLinear(d_model, 4 * d_model, device, seed + 3, gen, **more)
        self.fc_out = AnalogLinear(4 * d_model, d_model, device, seed + 4, gen, **more)

    def linears(self) -> List[AnalogLinear]:
        return [self.qkv, self.proj, self.fc, self.fc_out]

    def __call__(self, h: torch.Tensor, timer=None) -> torch.Tensor:
        b, s, d = h.shape
        a = F.layer_norm(h, (d,), self.ln1_w, self.ln1_b)
        q, k, v = timed(timer, self.qkv, a).split(d, dim=-1)
        shape = (b, s, self.n_head, d // self.n_head)
        q, k, v = (t.reshape(shape).transpose(1, 2) for t in (q, k, v))
        att = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        h = h + timed(timer, self.proj, att.transpose(1, 2).reshape(b, s, d))
        a = F.layer_norm(h, (d,), self.ln2_w, self.ln2_b)
        return h + timed(timer, self.fc_out, F.gelu(timed(timer, self.fc, a)))

    def adapted(self, a: torch.Tensor, h: torch.Tensor, next_norm, run: Adaptation, timer=None):
        """The block on its normalised input ``a`` and the residual stream ``h``; returns the same two for what follows,
        ``next_norm`` being the norm in front of that.  Each residual sum is one pass with its dropout and norm."""
        b, s, d = h.shape
        q, k, v = timed(timer, run.linear(self.qkv), a).split(d, dim=-1)
        shape = (b, s, self.n_head, d // self.n_head)
        q, k, v = (t.reshape(shape).transpose(1, 2) for t in (q, k, v))
        att = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        x = timed(timer, run.linear(self.proj), att.transpose(1, 2).reshape(b, s, d))
        a, h = run.add_norm(x, h, (self.ln2_w, self.ln2_b))
        x = timed(timer, run.linear(self.fc_out), F.gelu(timed(timer, run.linear(self.fc), a)))
        return run.add_norm(x, h, next_norm)


def timed(timer, fn, x):
    """Run ``fn(x)``; with a timer, bracket it with CUDA events on the current stream."""
    if timer is None:
        return fn(x)
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    y = fn(x)
    e1.record()
    timer.append((e0, e1))
    return y


class AnalogGPT2:
    def __init__(self, n_layer: int = 12, d_model: int = 768, n_head: int = 12, device: int = 0,
                 seed: int = 4, shard_tiles: bool = False, adapters: int = 0, rank: int = 16):
        gen = torch.Generator().manual_seed(seed)
        dev = f"cuda:{device}"
        self.device = dev
        self.d_model = d_model
        self.wte = (torch.randn(VOCAB, d_model, generator=gen) * 0.02).to(dev)
        self.wpe = (torch.randn(N_POS, d_model, generator=gen) * 0.01).to(dev)
        self.blocks = [Block(d_model, n_head, device, seed * 1000 + 10 * i, gen, shard_tiles, adapters, rank)
                       for i in range(n_layer)]
        self.lnf_w, self.lnf_b = torch.ones(d_model, device=dev), torch.zeros(d_model, device=dev)

    def forward(self, ids: torch.Tensor, timer=None, run: Optional[Adaptation] = None) -> torch.Tensor:
        """``ids`` [batch, seq] on the device -> id of the most likely next token per position."""
        b, s = ids.shape
        if run is not None:
            h = self.hidden(ids, run, timer)
        else:
            h = self.wte[ids] + self.wpe[:s]
            for blk in self.blocks:
                h = blk(h, timer)
            h = F.layer_norm(h, (self.d_model,), self.lnf_w, self.lnf_b)
        out = torch.empty(b, s, dtype=torch.long, device=ids.device)
        # vocabulary projection in row chunks: the full logits would be 3.3 GB per 16384 tokens
        flat = h.reshape(-1, self.d_model)
        chunk = 4096
        for r0 in range(0, flat.size(0), chunk):
            out.view(-1)[r0 : r0 + chunk] = (flat[r0 : r0 + chunk] @ self.wte.t()).argmax(dim=-1)
        return out

    def hidden(self, ids: torch.Tensor, run: Adaptation, timer=None) -> torch.Tensor:
        """Normalised output of the last block, with the adapters of ``run``."""
        from . import digital

        h = self.wte[ids] + self.wpe[: ids.size(1)]
        a = digital.layer_norm(h, self.blocks[0].ln1_w, self.blocks[0].ln1_b)
        for blk, after in zip(self.blocks, self.blocks[1:] + [None]):
            norm = (self.lnf_w, self.lnf_b) if after is None else (after.ln1_w, after.ln1_b)
            a, h = blk.adapted(a, h, norm, run, timer)
        return a

    def loss(self, ids: torch.Tensor, targets: torch.Tensor, run: Adaptation) -> torch.Tensor:
        """Mean cross entropy of the next tokens ``targets``."""
        logits = self.hidden(ids, run).reshape(-1, self.d_model) @ self.wte.t()
        return F.cross_entropy(logits, targets.reshape(-1))

    def trained(self) -> List[torch.Tensor]:
        """What adaptation changes: adapters and norms."""
        norms = [t for blk in self.blocks for t in (blk.ln1_w, blk.ln1_b, blk.ln2_w, blk.ln2_b)] + [self.lnf_w, self.lnf_b]
        return [q for blk in self.blocks for lin in blk.linears() for q in (lin.adapters.a, lin.adapters.b)] + norms

    def analog_flops_per_token(self) -> float:
        return sum(2.0 * lin.in_features * lin.out_features for blk in self.blocks for lin in blk.linears())

    def n_tiles(self) -> int:
        return sum(lin.n_tiles for blk in self.blocks for lin in blk.linears())


def sequence_adapters(first: int, count: int, n_adapters: int, device) -> torch.Tensor:
    """Adapters of the batch's sequences ``first``, ``first + 1``, ... (``count`` of them): in turn over the whole batch, however
    many ranks share it."""
    return torch.arange(first, first + count, device=device) % n_adapters


def adapt(model: AnalogGPT2, ids: torch.Tensor, n_adapters: int, steps: int, lr: float = 1e-3, p: float = 0.1) -> dict:
    """Training steps on the adapters and norms, one sequence at a time (the logits of one are 0.2 GB at 1024 tokens),
    gradients of the batch added up; returns the time of a step and the losses.  One process only: nothing here adds the
    gradients of several ranks up, and each would go on with a model of its own."""
    import torch.distributed as dist

    if dist.is_available() and dist.is_initialized() and dist.get_world_size() > 1:
        raise RuntimeError("adaptation runs in one process: gradients are not added up over ranks")
    if ids.size(1) < 2:
        raise RuntimeError("adaptation needs sequences of at least two tokens: the next one is what is learned")
    weights = model.trained()
    for t in weights:
        t.requires_grad_()
    opt = torch.optim.SGD(weights, lr=lr)
    losses, call = [], 0
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for step in range(steps):
        if step == min(1, steps - 1):
            e0.record()  # the first step allocates
        opt.zero_grad(set_to_none=True)
        total = torch.zeros((), device=ids.device)
        for j in range(ids.size(0)):
            run = Adaptation(torch.full((1,), j % n_adapters, device=ids.device), ids.size(1) - 1, p, seed=step, call=call)
            loss = model.loss(ids[j : j + 1, :-1], ids[j : j + 1, 1:], run) / ids.size(0)
            loss.backward()
            total += loss.detach()
            call = run.call
        opt.step()
        losses.append(total)
    e1.record()
    torch.cuda.synchronize()
    return {"ms_per_step": e0.elapsed_time(e1) / max(1, steps - 1), "steps": steps, "losses": [float(t) for t in losses]}


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=12)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--seq", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=5)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--shard", default="sequences", choices=["sequences", "tiles"],
                    help="N > 1: split the sequences over the ranks, or the tiles of every analog layer")
    ap.add_argument("--adapters", type=int, default=0, help="low-rank adapters beside every analog layer")
    ap.add_argument("--rank", type=int, default=16, help="rank of the adapters")
    ap.add_argument("--adapt-steps", type=int, default=0, help="training steps on adapters and norms after the forward passes (one process)")
    args = ap.parse_args(argv)
    world = int(os.environ.get("WORLD_SIZE", "1"))
    if args.adapt_steps and not args.adapters:
        raise SystemExit("--adapt-steps needs --adapters")
    if args.adapt_steps and world > 1:
        raise SystemExit("--adapt-steps runs in one process: gradients are not added up over ranks")
    if args.adapt_steps and args.seq < 2:
        raise SystemExit("--adapt-steps needs sequences of at least two tokens")

    import torch.distributed as dist

    from . import _cabi

    if not torch.cuda.is_available():
        raise RuntimeError("needs a CUDA device: the analog tiles have no CPU path")
    rank = int(os.environ.get("RANK", "0"))
    local_rank = int(os.environ.get("LOCAL_RANK", "0"))
    torch.cuda.set_device(local_rank)
    if world > 1:
        dist.init_process_group("nccl", device_id=torch.device("cuda", local_rank))
    shard_tiles = world > 1 and args.shard == "tiles"
    if args.batch % world and not shard_tiles:
        raise SystemExit("--batch must be a multiple of the number of ranks")
    local_batch = args.batch if shard_tiles else args.batch // world
    model = AnalogGPT2(args.layers, device=local_rank, seed=4, shard_tiles=shard_tiles, adapters=args.adapters,
                       rank=args.rank)
    k = 0
    for blk in model.blocks:  # independent noise per layer (and per rank when ranks hold replicas)
        for lin in blk.linears():
            lin.array.set_seed((1 if shard_tiles else 100003 * (rank + 1)) + k)
            k += 1
    g = torch.Generator().manual_seed(4 + (0 if shard_tiles else rank))
    ids_host = torch.randint(0, VOCAB, (local_batch, args.seq), generator=g).pin_memory()
    out_host = torch.empty(local_batch, args.seq, dtype=torch.long).pin_memory()
    ids = ids_host.to(model.device)
    run = None
    if args.adapters:
        run = Adaptation(sequence_adapters(rank * local_batch, local_batch, args.adapters, model.device), args.seq)

    def barrier():
        if world > 1:
            dist.barrier()
        torch.cuda.synchronize()

    def timed_loop(fn, steps):
        barrier()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(steps):
            fn()
        e1.record()
        barrier()
        ms = torch.tensor([e0.elapsed_time(e1)], device=model.device)
        if world > 1:
            dist.all_reduce(ms, op=dist.ReduceOp.MAX)
        return float(ms) / steps

    with torch.no_grad():
        for _ in range(args.warmup):
            model.forward(ids, run=run)
        launches0 = _cabi.lib().ab200_kernel_launch_count()
        ms = timed_loop(lambda: model.forward(ids, run=run), args.steps)
        launches = (_cabi.lib().ab200_kernel_launch_count() - launches0) // args.steps

        def e2e():
            d = ids_host.to(model.device, non_blocking=True)
            out_host.copy_(model.forward(d, run=run), non_blocking=True)

        e2e()
        ms_e2e = timed_loop(e2e, args.steps)
        timer = []
        torch.cuda.synchronize()
        model.forward(ids, timer, run)
        torch.cuda.synchronize()
        analog_ms = sum(a.elapsed_time(b) for a, b in timer)
    adaptation = adapt(model, ids, args.adapters, args.adapt_steps) if args.adapt_steps else None
    tokens = args.batch * args.seq
    if rank == 0:
        flops = model.analog_flops_per_token() * local_batch * args.seq / (world if shard_tiles else 1)
        print(json.dumps({
            "metric": "analog_inference_tokens_per_s", "value": tokens / (ms * 1e-3), "unit": "tokens/s",
            "n_gpus": world, "steps": args.steps, "warmup": args.warmup, "ms_per_step": ms,
            "higher_is_better": True, "scaling": "strong", "dtype": "f32 (analog layers: DAC codes x split-bf16 weights, f32 accumulate)",
            "data": "synthetic",
            "config": {"workload": f"GPT-2-small-shaped forward, {args.layers} blocks, batch {args.batch} x seq {args.seq}",
                       "analog_tiles": model.n_tiles(), "parallelism": (f"tiles of every analog layer over {world} rank(s), all-reduce of the "
                                       "partial outputs, digital parts replicated" if shard_tiles
                                       else f"sequences over {world} rank(s)")},
            "e2e": {"value": tokens / (ms_e2e * 1e-3), "unit": "tokens/s",
                    "h2d_bytes_per_step": ids_host.numel() * 8 * (1 if shard_tiles else world),
                    "d2h_bytes_per_step": out_host.numel() * 8 * (1 if shard_tiles else world)},
            "analog_layers": {"ms_per_step": analog_ms, "share": analog_ms / ms,
                              "logical_tflops": flops / (analog_ms * 1e-3) / 1e12},
            "gpu_launches": int(launches),
            **({"adapters": {"count": args.adapters, "rank": args.rank}} if args.adapters else {}),
            **({"adaptation": adaptation} if adaptation else {}),
        }))
    if world > 1:
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
