"""Trains a small model on its resident state, through a switch of its parallel layout.

    python examples/train_through_switch.py [--steps 12] [--switch-at 6]

Every rank's state lives on one GPU, as the resharding manager holds it.  A step runs the model forward and
backward (plain torch; the loss over the output layer's vocabulary shards as the state holds them is
``training.linear_cross_entropy``), then updates the state: ``training.muon_step`` on the matrices of the
layers, gathered from their shards, ``training.adamw_step`` on every rank's own shard of the rest.  In the
middle the job switches from TP1 to TP2 with ``ElasticMegatronManager.reshard``, and training goes on.
"""

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from elasticmegatron_amd import ElasticMegatronManager, ModelSpec, training  # noqa: E402
from elasticmegatron_amd.resharding.layout import geometry  # noqa: E402

BEFORE = dict(world_size=4, tensor_model_parallel_size=1, pipeline_model_parallel_size=1)
AFTER = dict(world_size=4, tensor_model_parallel_size=2, pipeline_model_parallel_size=1)


def small_model() -> ModelSpec:
    return ModelSpec(name="small", num_layers=2, hidden_size=128, num_attention_heads=4, ffn_hidden_size=344,
                     padded_vocab_size=1024, vocab_size=1000, overlap_grad_reduce=False)


class Parameters:
    """A state's parameters as whole tensors: gathered from the ranks' shards and put back."""

    def __init__(self, state, space):
        self.state, self.layout, self.params = state, state.layout, space.all_virtual_params

    def _parts(self, vp, whole):
        """(TP rank, local rows, their place in ``whole``) of every shard of ``vp``."""
        tp = self.layout.strategy.tensor_model_parallel_size
        for t in range(tp):
            g = geometry(vp, tp, t)
            for lo, hi, row in g.bands():
                yield t, slice(lo, hi), whole[row:row + hi - lo, g.col_off:g.col_off + g.cols]

    def _two_d(self, vp):
        g = geometry(vp, 1, 0)
        return g.rows, g.cols

    def _local(self, vp):
        g = geometry(vp, self.layout.strategy.tensor_model_parallel_size, 0)
        return g.rows, g.cols

    def gather(self, vp, arena):
        """The whole of ``vp`` from an fp32 arena (every rank's flat shard) or from the bf16 arena."""
        holders = self.layout.bf16_holders(vp) if arena.dtype == torch.bfloat16 else self.layout.fp32_holders(vp)
        rows, cols = self._local(vp)
        tp = self.layout.strategy.tensor_model_parallel_size
        local = [torch.empty(rows * cols, dtype=arena.dtype, device=arena.device) for _ in range(tp)]
        for h in holders:
            local[h.tp_rank][h.lo:h.hi] = arena[h.offset:h.offset + h.hi - h.lo]
        whole = torch.empty(self._two_d(vp), dtype=arena.dtype, device=arena.device)
        for t, part, place in self._parts(vp, whole):
            place.copy_(local[t].view(rows, cols)[part])
        return whole.view(vp.full_shape)

    def local_parts(self, vp, whole):
        """``whole`` as every TP rank's local tensor, flat."""
        rows, cols = self._local(vp)
        tp = self.layout.strategy.tensor_model_parallel_size
        local = [torch.empty(rows, cols, dtype=whole.dtype, device=whole.device) for _ in range(tp)]
        for t, part, place in self._parts(vp, whole.view(self._two_d(vp))):
            local[t][part] = place
        return [x.view(-1) for x in local]

    def put(self, vp, whole, arena):
        local = self.local_parts(vp, whole)
        holders = self.layout.bf16_holders(vp) if arena.dtype == torch.bfloat16 else self.layout.fp32_holders(vp)
        for h in holders:
            arena[h.offset:h.offset + h.hi - h.lo] = local[h.tp_rank][h.lo:h.hi]

    def initialise(self, seed):
        gen = torch.Generator(device=self.state.device).manual_seed(seed)
        for vp in self.params:
            shape = vp.full_shape
            if len(shape) == 1:
                w = torch.ones(shape, device=self.state.device)
            else:
                w = torch.randn(shape, generator=gen, device=self.state.device) * 0.02
            self.put(vp, w, self.state.main)
            self.put(vp, w.to(torch.bfloat16), self.state.param)
        self.state.exp_avg.zero_()
        self.state.exp_avg_sq.zero_()


def is_matrix_of_a_layer(vp):
    return len(vp.full_shape) == 2 and "embedding" not in vp.param_def.name and "output_layer" not in vp.param_def.name


def rms_norm(x, weight):
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-5) * weight.float()).to(x.dtype)


def attention(x, qkv, proj, heads):
    b, n, h = x.shape
    q, k, v = (x @ qkv.t()).view(b, n, heads, 3, h // heads).float().permute(3, 0, 2, 1, 4).contiguous().unbind(0)
    scores = (q @ k.transpose(-1, -2).contiguous()) / math.sqrt(h // heads)
    scores = scores.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf)
    out = (scores.softmax(-1) @ v).to(x.dtype)
    return out.transpose(1, 2).reshape(b, n, h) @ proj.t()


def hidden_states(spec, weights, tokens):
    x = weights["embedding.word_embeddings.weight"][tokens]
    for layer in range(spec.num_layers):
        w = lambda name: weights[f"{layer}.{name}"]  # noqa: E731
        y = rms_norm(x, w("self_attention.linear_qkv.layer_norm_weight"))
        x = x + attention(y, w("self_attention.linear_qkv.weight"), w("self_attention.linear_proj.weight"), spec.num_attention_heads)
        y = rms_norm(x, w("mlp.linear_fc1.layer_norm_weight")) @ w("mlp.linear_fc1.weight").t()
        gate, up = y.chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w("mlp.linear_fc2.weight").t()
    return rms_norm(x, weights["decoder.final_layernorm.weight"])


def key_of(vp):
    layer = vp.param_position_attr.transformer_layer_id  # -1: not of a layer
    return vp.param_def.name if layer < 0 else f"{layer}.{vp.param_def.name}"


def train_step(spec, params, tokens, targets, step, lr=2e-3):
    """One step on the state; returns the loss."""
    state = params.state
    output = next(vp for vp in params.params if vp.param_def.name == "output_layer.weight")
    tp = state.layout.strategy.tensor_model_parallel_size
    weights = {key_of(vp): params.gather(vp, state.param).requires_grad_() for vp in params.params if vp is not output}
    shards = [state.model_param(output, t).detach().requires_grad_() for t in range(tp)]  # as the state holds them
    loss = training.linear_cross_entropy(hidden_states(spec, weights, tokens), shards, targets, vocab_size=spec.vocab_size)
    loss.backward()
    for vp in params.params:
        if is_matrix_of_a_layer(vp):
            main, momentum = params.gather(vp, state.main), params.gather(vp, state.exp_avg)
            image = torch.empty_like(main, dtype=torch.bfloat16)
            training.muon_step(main, momentum, weights[key_of(vp)].grad, model=image, lr=lr, weight_decay=0.01)
            for whole, arena in ((main, state.main), (momentum, state.exp_avg), (image, state.param)):
                params.put(vp, whole, arena)
            continue
        local = [s.grad.view(-1) for s in shards] if vp is output else params.local_parts(vp, weights[key_of(vp)].grad)
        images = {h.tp_rank: h.offset for h in state.layout.bf16_holders(vp)}
        for h in state.layout.fp32_holders(vp):  # every rank its own shard
            own = slice(h.offset, h.offset + h.hi - h.lo)
            image = state.param[images[h.tp_rank] + h.lo:images[h.tp_rank] + h.hi]
            training.adamw_step(state.main[own], state.exp_avg[own], state.exp_avg_sq[own], local[h.tp_rank][h.lo:h.hi], model=image, lr=lr,
                                weight_decay=0.01, step=step)
    return float(loss.detach())


def run(steps, switch_at, seed=7, device="cuda:0"):
    """The losses of ``steps`` steps, with the switch after ``switch_at`` of them (never: None)."""
    spec = small_model()
    mgr = ElasticMegatronManager([BEFORE, AFTER], spec, device=device, release_source=False)
    params = Parameters(mgr.training_state, mgr.virtual_param_space)
    params.initialise(seed)
    gen = torch.Generator(device=device).manual_seed(seed)
    text = torch.randint(0, spec.vocab_size, (8, 65), generator=gen, device=device)
    targets = text[:, 1:].clone()
    targets[:, :4] = -100  # the prompt's tokens do not count
    losses = []
    for step in range(steps):
        if step == switch_at:
            before = params
            mgr.reshard(new_parallel_strategy=AFTER)
            params = Parameters(mgr.training_state, mgr.virtual_param_space)
            for vp in params.params:  # the same bits, in another layout
                for kind in ("main", "exp_avg", "exp_avg_sq", "param"):
                    assert torch.equal(params.gather(vp, getattr(params.state, kind)), before.gather(vp, getattr(before.state, kind)))
        losses.append(train_step(spec, params, text[:, :-1], targets, step + 1))
    return losses


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=12)
    ap.add_argument("--switch-at", type=int, default=6)
    args = ap.parse_args()
    for step, (with_switch, without) in enumerate(zip(run(args.steps, args.switch_at), run(args.steps, None))):
        print(f"step {step}: loss {with_switch:.6f}, without the switch {without:.6f}" + ("  <- switched before" if step == args.switch_at else ""))


if __name__ == "__main__":
    main()
