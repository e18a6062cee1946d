"""The operators of a training step over the resident state, as cases that a timing program can run.

``score``        the loss of every token from the output layer's weight, with no gradient: log-probabilities
                 of given tokens, from a single one
``loss``         the same loss with its gradients to the hidden states and to every vocabulary shard
``orthogonalise``  Newton-Schulz products on one matrix or on several of one shape
``muon``         the whole Muon update of such matrices: momentum, Newton-Schulz, decayed weights, bf16 image
``adamw``        the AdamW update of what Muon does not train (embeddings, output layer, norms)

Sizes are those of the models this framework reshards (tiny LLaMA-2, Llama-2-7B, Llama-3-8B, the ragged
test model) and of nothing in particular.  The plain forms are elementary torch operations in 32 bits.
"""

import math

import torch

own = False

IGNORED = -100
MUON = dict(lr=3e-4, momentum=0.95, weight_decay=0.1, rms_scale=0.2)
ADAM = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=100)
A, B, C = 3.4445, -4.7750, 2.0315
STEPS = 5
EPS = 1e-7


def _ce(mode, tokens, hidden, vocab, padded=0, shards=1, dtype="bf16"):
    """``vocab`` rows that count, of ``padded`` rows cut into ``shards`` equal tensor-parallel shards."""
    return dict(op=mode, tokens=tokens, hidden=hidden, vocab=vocab, padded=padded or vocab, shards=shards, dtype=dtype)


def _matrices(op, count, rows, cols, grad="fp32"):
    return dict(op=op, count=count, rows=rows, cols=cols, grad=grad)


def _adamw(numel, grad="fp32", model=True):
    return dict(op="adamw", numel=numel, grad=grad, model=model)


def listed():
    return [
        # The log-probability of one token under Llama-2-7B's output layer: one pass over its weight.
        dict(_ce("score", 1, 4096, 32000), name="score-one-token"),
        # A ragged batch scored by the ragged test model: a hidden size that fills no tile, in fp16.
        dict(_ce("score", 333, 1000, 32000, dtype="fp16"), name="score-ragged"),
        # One training step of the tiny LLaMA-2 of the demo, its vocabulary cut by TP4.
        dict(_ce("loss", 500, 512, 32000, shards=4), name="loss-tiny-tp4"),
        # A micro-batch of Llama-2-7B: 4096 tokens.
        dict(_ce("loss", 4096, 4096, 32000), name="loss-7b"),
        # Llama-3-8B with its vocabulary padded for TP4, whose last shard holds rows that do not count.
        dict(_ce("loss", 4096, 4096, 128256, padded=128512, shards=4), name="loss-llama3-tp4-padded"),
        # The smallest update that Muon sees here: the two projections of a unit test's model.
        dict(_matrices("orthogonalise", 2, 128, 128), name="orth-smallest"),
        # A stack of the ragged model's FFN matrices, bf16 gradients.
        dict(_matrices("orthogonalise", 8, 2668, 1000, grad="bf16"), name="orth-ragged-stack"),
        # The tiny LLaMA-2's two FFN output matrices.
        dict(_matrices("muon", 2, 512, 1376), name="muon-tiny"),
        # Llama-2-7B's attention output projections of four layers.
        dict(_matrices("muon", 4, 4096, 4096), name="muon-7b-proj"),
        # Its fused gate and up projection of one layer, the largest matrix of a layer; bf16 gradients.
        dict(_matrices("muon", 1, 22016, 4096, grad="bf16"), name="muon-7b-fc1"),
        # The norm weights of a small model: latency is all of it.
        dict(_adamw(4 * 1000 + 1), name="adamw-norms"),
        # Llama-2-7B's embedding.
        dict(_adamw(32000 * 4096, grad="bf16"), name="adamw-embedding"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "loss", "loss", "orthogonalise", "muon", "muon", "adamw"])
    if op in ("score", "loss"):
        shards = rng.choice([1, 1, 2, 4])
        tokens = _log_uniform(rng, 1, 4096)
        hidden = rng.choice([128, 256, 512, 1000, 1024, 2048, 4096, 8 * rng.randrange(16, 512) + rng.choice([0, 0, 0, 4, 1])])
        rows = -(-_log_uniform(rng, 512, 128256) // shards)
        padded = rows * shards
        return _ce(op, tokens, 4104 if hidden == 3072 else hidden, padded - rng.choice([0, 0, rng.randrange(1, rows // 2)]), padded,
                   shards, rng.choice(["bf16", "bf16", "bf16", "fp16"]))
    if op == "adamw":
        return _adamw(_log_uniform(rng, 1, 32000 * 4096), rng.choice(["fp32", "bf16"]), rng.random() < 0.7)
    rows = _log_uniform(rng, 16, 4096)
    cols = min(22016, max(8, int(rows * math.exp(rng.uniform(-0.2, 1.7)))))
    if rng.random() < 0.4:
        rows, cols = -(-rows // 64) * 64, -(-cols // 64) * 64
    rows, cols = (1 + x if x == 3072 else x for x in (rows, cols))
    if rng.random() < 0.5:
        rows, cols = cols, rows
    count = rng.choice([1, 2, 3, 4, 8]) if rows * cols < 4096 * 4096 else 1
    return _matrices(op, count, rows, cols, rng.choice(["fp32", "bf16"]))


DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gradients(case, gen):
    """Gradients as training makes them: a few strong directions that fall off, over noise."""
    n, m, k = case["count"], case["rows"], case["cols"]
    r = min(64, m, k)
    u = torch.randn(n, m, r, generator=gen, device="cuda") / torch.arange(1, r + 1, device="cuda")
    v = torch.randn(n, r, k, generator=gen, device="cuda")
    g = torch.baddbmm(torch.randn(n, m, k, generator=gen, device="cuda"), u, v, beta=0.1)
    return g.mul_(1e-3).to(DTYPES[case["grad"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = dict(generator=gen, device="cuda")
    op = case["op"]
    if op in ("score", "loss"):
        t, h, dt = case["tokens"], case["hidden"], DTYPES[case["dtype"]]
        weight = torch.randn(case["padded"], h, **dev) / math.sqrt(h)
        target = torch.randint(0, case["vocab"], (t,), **dev)
        # Normalised hidden states that lean towards their token's row, as a trained model's do: the
        # target's logit is about 4 where the others spread by 1.
        hidden = torch.randn(t, h, **dev) + 4 * weight[target]
        if t > 1:
            target[torch.rand(t, **dev) < 0.1] = IGNORED
        state = dict(case, hidden=hidden.to(dt), target=target,
                     shards=[w.contiguous() for w in weight.to(dt).chunk(case["shards"])])
        if op == "loss":
            # Each token's share of the step's loss: packed documents count by their length.
            state["grad_loss"] = (0.5 + torch.rand(t, **dev)) / t
            state["hidden"].requires_grad_()
            for w in state["shards"]:
                w.requires_grad_()
        return state
    if op == "adamw":
        n = case["numel"]
        g = (torch.randn(n, **dev) * 1e-3).to(DTYPES[case["grad"]])
        return dict(case, main=torch.randn(n, **dev) * 0.02, exp_avg=torch.randn(n, **dev) * 3e-4,
                    exp_avg_sq=(torch.randn(n, **dev) * 1e-3).square_(), grad=g,
                    image=torch.empty(n, dtype=torch.bfloat16, device="cuda") if case["model"] else None)
    grad = _gradients(case, gen)
    if op == "orthogonalise":
        return dict(case, grad=grad)
    n, m, k = case["count"], case["rows"], case["cols"]
    return dict(case, grad=grad, main=torch.randn(n, m, k, **dev) * 0.02,
                momentum=_gradients(dict(case, grad="fp32"), gen).mul_(5),
                image=torch.empty(n, m, k, dtype=torch.bfloat16, device="cuda"))


# ----- the plain forms -----


def _plain_loss(s, grads):
    hidden, target = s["hidden"].detach().float(), s["target"]
    weight = torch.cat([w.detach() for w in s["shards"]]).float()
    logits = hidden @ weight.t()
    logits[:, s["vocab"]:] = -math.inf
    top = logits.amax(1, keepdim=True)
    e = (logits - top).exp()
    total = e.sum(1, keepdim=True)
    lse = top + total.log()
    counts = target != IGNORED
    at = torch.where(counts, target, 0)[:, None]
    loss = torch.where(counts, (lse - logits.gather(1, at))[:, 0], 0.0)
    if not grads:
        return loss
    scale = torch.where(counts, s["grad_loss"], 0.0)[:, None]
    d = e * (scale / total)
    d.scatter_add_(1, at, -scale)
    dt = s["hidden"].dtype
    return [loss, (d @ weight).to(dt), *(d.t() @ hidden).to(dt).chunk(s["shards_n"])]


def _plain_orthogonalise(g):
    x = g.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2).contiguous()
        x = A * x + (B * gram + C * (gram @ gram)) @ x
    return x.transpose(1, 2) if tall else x


def _plain_muon(s):
    main, buf, g = s["main"], s["momentum"], s["grad"].float()
    buf.mul_(MUON["momentum"]).add_(g)
    o = _plain_orthogonalise(g + MUON["momentum"] * buf)
    main.mul_(1 - MUON["lr"] * MUON["weight_decay"])
    main.sub_(o * (MUON["lr"] * MUON["rms_scale"] * math.sqrt(max(s["rows"], s["cols"]))))
    s["image"].copy_(main)
    return [main, buf, s["image"]]


def _plain_adamw(s):
    main, m, v, g = s["main"], s["exp_avg"], s["exp_avg_sq"], s["grad"].float()
    m.mul_(ADAM["beta1"]).add_(g * (1 - ADAM["beta1"]))
    v.mul_(ADAM["beta2"]).add_(g * g * (1 - ADAM["beta2"]))
    m_hat = m / (1 - ADAM["beta1"] ** ADAM["step"])
    v_hat = v / (1 - ADAM["beta2"] ** ADAM["step"])
    main.mul_(1 - ADAM["lr"] * ADAM["weight_decay"])
    main.sub_(ADAM["lr"] * m_hat / (v_hat.sqrt() + ADAM["eps"]))
    if s["image"] is None:
        return [main, m, v]
    s["image"].copy_(main)
    return [main, m, v, s["image"]]


def _plain(s):
    op = s["op"]
    if op in ("score", "loss"):
        return _plain_loss(dict(s, shards_n=len(s["shards"])), op == "loss")
    if op == "orthogonalise":
        return _plain_orthogonalise(s["grad"]).to(torch.bfloat16).contiguous()
    return _plain_muon(s) if op == "muon" else _plain_adamw(s)


# ----- the framework's calls -----


def _framework(s):
    from elasticmegatron_amd import training

    op = s["op"]
    if op in ("score", "loss"):
        loss = training.linear_cross_entropy(s["hidden"], s["shards"], s["target"], vocab_size=s["vocab"],
                                             ignore_index=IGNORED, reduction="none")
        if op == "score":
            return loss
        return [loss, *torch.autograd.grad(loss, [s["hidden"], *s["shards"]], s["grad_loss"])]
    if op == "orthogonalise":
        return training.orthogonalise(s["grad"], steps=STEPS, coefficients=(A, B, C), eps=EPS)
    if op == "muon":
        training.muon_step(s["main"], s["momentum"], s["grad"], model=s["image"], steps=STEPS, coefficients=(A, B, C),
                           eps=EPS, nesterov=True, **MUON)
        return [s["main"], s["momentum"], s["image"]]
    training.adamw_step(s["main"], s["exp_avg"], s["exp_avg_sq"], s["grad"], model=s["image"], **ADAM)
    return [s["main"], s["exp_avg"], s["exp_avg_sq"]] + ([] if s["image"] is None else [s["image"]])


def run(state):
    return _framework(state) if own else _plain(state)


# ----- what they cannot do without -----


def work(case):
    op = case["op"]
    if op in ("score", "loss"):
        t, h, v = case["tokens"], case["hidden"], case["padded"]
        read = 2 * (t + v) * h + 8 * t
        if op == "score":
            return {"bytes": read + 4 * t, "flops": 2 * t * h * v}
        return {"bytes": read + 4 * t + 2 * (t + v) * h + 4 * t, "flops": 6 * t * h * v}
    if op == "adamw":
        n = case["numel"]
        return {"bytes": n * (24 + (4 if case["grad"] == "fp32" else 2) + (2 if case["model"] else 0)), "flops": 16 * n}
    n, short, long = case["count"], *sorted((case["rows"], case["cols"]))
    # A step: the Gram matrix and its square are symmetric, so that half of each is enough.
    flops = n * STEPS * (3 * short * short * long + short ** 3)
    g = 4 if case["grad"] == "fp32" else 2
    return {"bytes": n * short * long * (g + (2 if op == "orthogonalise" else 18)), "flops": flops}


# ----- 64 bits, from the definitions -----


def _exact_newton_schulz(g):
    out = []
    for x in g.double():
        wide = x if x.shape[0] <= x.shape[1] else x.t().contiguous()
        wide = wide / (torch.linalg.matrix_norm(wide) + EPS)
        for _ in range(STEPS):
            gram = wide @ wide.t()
            p = torch.addmm(gram, gram, gram, beta=B, alpha=C)
            p.diagonal().add_(A)
            wide = p @ wide
        out.append(wide if x.shape[0] <= x.shape[1] else wide.t())
    return torch.stack(out)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("score", "loss"):
        hidden = s["hidden"].detach().double()
        shards = [w.detach().double() for w in s["shards"]]
        logits = torch.cat([hidden @ w.t() for w in shards], 1)[:, :case["vocab"]]
        logp = torch.log_softmax(logits, 1)
        loss = torch.nn.functional.nll_loss(logp, s["target"], ignore_index=IGNORED, reduction="none")
        if op == "score":
            return loss
        del logits
        d = logp.exp_()
        rows = torch.arange(case["tokens"], device="cuda")[s["target"] != IGNORED]
        d[rows, s["target"][rows]] -= 1.0
        d *= (s["grad_loss"].double() * (s["target"] != IGNORED))[:, None]
        dh, dw, lo = torch.zeros_like(hidden), [], 0
        for w in shards:
            part = d[:, lo:lo + w.shape[0]]
            dh += part @ w[:part.shape[1]]
            dw.append(torch.zeros_like(w))
            dw[-1][:part.shape[1]] = part.t() @ hidden
            lo += w.shape[0]
        return [loss, dh, *dw]
    if op == "orthogonalise":
        return _exact_newton_schulz(s["grad"])
    g, main = s["grad"].double(), s["main"].double()
    if op == "muon":
        buf = MUON["momentum"] * s["momentum"].double() + g
        o = _exact_newton_schulz(g + MUON["momentum"] * buf)
        main = main * (1 - MUON["lr"] * MUON["weight_decay"]) - MUON["lr"] * MUON["rms_scale"] * max(main.shape[1:]) ** 0.5 * o
        return [main, buf, main]
    m = torch.lerp(g, s["exp_avg"].double(), ADAM["beta1"])
    v = torch.lerp(g ** 2, s["exp_avg_sq"].double(), ADAM["beta2"])
    hat = m / (1 - ADAM["beta1"] ** ADAM["step"]) / ((v / (1 - ADAM["beta2"] ** ADAM["step"])) ** 0.5 + ADAM["eps"])
    main = main - ADAM["lr"] * (ADAM["weight_decay"] * main + hat)
    return [main, m, v] + ([main] if case["model"] else [])
