"""A layer of a mixture of experts, and the loss behind it, from the operators of a training step together."""

import math

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, HIDDEN, FFN, EXPERTS, TOP, VOCAB = 8, 2, 32, 256, 344, 4, 2, 500
LENGTHS = [70, 1, 0, 129, 56]
BF16 = torch.bfloat16


def _weights(gen):
    r = lambda *s, scale=1.0: torch.randn(*s, generator=gen, device="cuda") * scale  # noqa: E731
    w = dict(norm1=1 + 0.1 * r(HIDDEN), qkv=r((HEADS + 2 * KV_HEADS) * DIM, HIDDEN, scale=HIDDEN ** -0.5), proj=r(HIDDEN, HEADS * DIM, scale=0.1),
             after=1 + 0.1 * r(HIDDEN), gate=0.5 + 0.1 * r(HIDDEN), norm2=1 + 0.1 * r(HIDDEN), norm3=1 + 0.1 * r(HIDDEN),
             out=r(VOCAB, HIDDEN, scale=HIDDEN ** -0.5))
    for e in range(EXPERTS):
        w[f"fc1.{e}"], w[f"fc2.{e}"] = r(2 * FFN, HIDDEN, scale=HIDDEN ** -0.5), r(HIDDEN, FFN, scale=FFN ** -0.5)
    return {k: v.to(BF16) for k, v in w.items()}


def _route(tokens, gen):
    """Two experts for every token, one expert with none, and their shares: what a router leaves."""
    experts = torch.stack([torch.randperm(EXPERTS - 1, generator=gen, device="cuda")[:TOP] for _ in range(tokens)])
    share = torch.rand(tokens, TOP, generator=gen, device="cuda").softmax(1)
    order = experts.flatten().argsort(stable=True)
    return order, order // TOP, torch.bincount(experts.flatten(), minlength=EXPERTS), share.flatten()[order]


def _own(x, w, route, offsets, target):
    order, token, counts, share = route
    y = training.rms_norm(x, w["norm1"])
    qkv = (y @ w["qkv"].t()).view(-1, HEADS + 2 * KV_HEADS, DIM)
    a = training.attention(qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:], offsets=offsets)
    x, y = training.residual_norm(x, a.flatten(1) @ w["proj"].t(), w["norm2"], branch_weight=w["after"], gate=w["gate"])
    h = training.expert_linear(y[token], [w[f"fc1.{e}"] for e in range(EXPERTS)], counts)
    gate, up = h.chunk(2, 1)
    z = training.expert_linear(torch.nn.functional.silu(gate) * up, [w[f"fc2.{e}"] for e in range(EXPERTS)], counts)
    z = torch.zeros_like(y).index_add_(0, token, z * share[:, None].to(BF16))
    _, y = training.residual_norm(x, z, w["norm3"], residual_scale=0.9)
    return training.linear_cross_entropy(y, w["out"], target)


def _plain(x, w, route, target):
    order, token, counts, share = route
    norm = lambda t, g: t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt() * g  # noqa: E731
    y = norm(x, w["norm1"])
    qkv = (y @ w["qkv"].t()).view(-1, HEADS + 2 * KV_HEADS, DIM)
    out, lo = [], 0
    for n in LENGTHS:
        q, k, v = (t.transpose(0, 1) for t in qkv[lo:lo + n].split([HEADS, KV_HEADS, KV_HEADS], 1))
        s = q @ k.repeat_interleave(HEADS // KV_HEADS, 0).transpose(1, 2) / math.sqrt(DIM)
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf)
        out.append((s.softmax(2) @ v.repeat_interleave(HEADS // KV_HEADS, 0)).transpose(0, 1).reshape(n, HEADS * DIM))
        lo += n
    x = x + w["gate"] * norm(torch.cat(out) @ w["proj"].t(), w["after"])
    y = norm(x, w["norm2"])[token]
    parts, lo = [], 0
    for e, n in enumerate(counts.tolist()):
        gate, up = (y[lo:lo + n] @ w[f"fc1.{e}"].t()).chunk(2, 1)
        parts.append((torch.nn.functional.silu(gate) * up) @ w[f"fc2.{e}"].t())
        lo += n
    x = 0.9 * x + torch.zeros_like(x).index_add(0, token, torch.cat(parts) * share[:, None])
    return torch.nn.functional.cross_entropy(norm(x, w["norm3"]) @ w["out"].t(), target)


def test_a_layer_of_experts(gpu_device):
    gen = torch.Generator(device="cuda").manual_seed(11)
    tokens = sum(LENGTHS)
    w = _weights(gen)
    x = torch.randn(tokens, HIDDEN, generator=gen, device="cuda").to(BF16)
    target = torch.randint(0, VOCAB, (tokens,), generator=gen, device="cuda")
    route = _route(tokens, gen)
    offsets = torch.tensor([0, *torch.tensor(LENGTHS).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    leaves = {"x": x, **w}
    own = {k: v.detach().requires_grad_() for k, v in leaves.items()}
    loss = _own(own["x"], own, route, offsets, target)
    got = dict(zip(own, torch.autograd.grad(loss, list(own.values()), materialize_grads=True)))
    exact = {k: v.detach().double().cpu().requires_grad_() for k, v in leaves.items()}
    cpu = [t.cpu() for t in route]
    want_loss = _plain(exact["x"], exact, [*cpu[:3], cpu[3].double()], target.cpu())
    want = dict(zip(exact, torch.autograd.grad(want_loss, list(exact.values()), materialize_grads=True)))
    # Forward, a value passes 16 roundings to bf16 on its longest way (norm, qkv, probabilities, out, proj, stream, norm, fc1, silu, product, fc2, share
    # and its product, sum over two experts, stream, norm), and as many backward: each moves it by 2^-8 of itself at most, and what it
    # depends on by as much, through functions whose slopes are about one.
    assert abs(float(loss) - float(want_loss)) <= 16 * 2.0 ** -8 * abs(float(want_loss))
    for k, g in got.items():
        off = (g.double().cpu() - want[k]).norm() / max(float(want[k].norm()), 1e-30)
        assert off <= 32 * 2.0 ** -8, (k, float(off))
    assert not got[f"fc1.{EXPERTS - 1}"].any() and not got[f"fc2.{EXPERTS - 1}"].any()  # the expert without tokens
