"""The operators of a training step's layers, as cases that a timing program can run.

``norm``       a block's output into the residual stream (through its own norm, a gate and a residual scale, as
               far as the case has them) and the norm before the next block
``experts``    products of every token with its expert's weight matrix, over experts of ragged sizes
``attention``  attention within packed documents, or of the last queries to longer keys

``train`` cases return the gradients of every input too.  Sizes are those of the models this framework
reshards (tiny LLaMA-2, Llama-2-7B and 70B, Llama-3-8B, Mixtral 8x7B, the ragged test model) and of nothing
in particular.  The plain forms are elementary torch operations in 32 bits.
"""

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _norm(tokens, hidden, dtype="bf16", residual=None, branch_norm=False, gate="none", scale=1.0, train=True):
    """``residual``: the stream's type; ``gate``: none, one for each channel, or one for each token's channels."""
    return dict(op="norm", tokens=tokens, hidden=hidden, dtype=dtype, residual=residual or dtype, branch_norm=branch_norm,
                gate=gate, scale=scale, train=train)


def _experts(counts, n_in, n_out, dtype="bf16", spare=0, train=True):
    """``counts``: tokens of each expert, as a text; ``spare``: rows behind the last expert's."""
    return dict(op="experts", counts=",".join(map(str, counts)), n_in=n_in, n_out=n_out, dtype=dtype, spare=spare, train=train)


def _attention(queries, heads, kv_heads, dim, keys=None, dtype="bf16", causal=True, spare=0, train=True):
    """``queries``, ``keys``: lengths of the documents, as a text; ``spare``: rows behind the last document."""
    return dict(op="attention", queries=",".join(map(str, queries)), keys=",".join(map(str, keys or queries)), heads=heads,
                kv_heads=kv_heads, dim=dim, dtype=dtype, causal=causal, spare=spare, train=train)


def listed():
    return [
        # A micro-batch of the tiny LLaMA-2 of the demo: latency is most of it.
        dict(_norm(500, 512), name="norm-tiny"),
        # The ragged test model in fp16, a gate for every token: rows that fill no wavefront.
        dict(_norm(333, 1000, "fp16", branch_norm=True, gate="token", scale=0.5), name="norm-ragged-token-gate"),
        # Llama-2-7B, 4096 tokens: a residual connection and the norm behind it.
        dict(_norm(4096, 4096), name="norm-7b"),
        # Llama-2-70B's width with the stream in 32 bits, norms on both sides of the block and a scale for each channel.
        dict(_norm(8192, 8192, residual="fp32", branch_norm=True, gate="channel", scale=0.9), name="norm-70b-sandwich"),
        # One token of Mixtral, top 2 of 8: two experts' first matrices read once.
        dict(_experts([0, 1, 0, 0, 0, 1, 0, 0], 4096, 28672, train=False), name="experts-one-token"),
        # A small mixture in fp16 with an expert that got nothing and spare rows: sizes that fill no tile.
        dict(_experts([41, 0, 97, 1, 64, 30, 15, 85], 1000, 2668, "fp16", spare=19), name="experts-ragged"),
        # Mixtral's second matrices on one rank of EP4: two experts, 4096 tokens of the batch between them.
        dict(_experts([2330, 1766], 14336, 4096), name="experts-mixtral-fc2-ep4"),
        # Mixtral's fused gate and up matrices, all 8 experts, 4096 tokens to two experts each.
        dict(_experts([1310, 745, 1024, 1398, 602, 1121, 893, 1099], 4096, 28672), name="experts-mixtral-fc1"),
        # The tiny LLaMA-2: short packed documents, one of them empty.
        dict(_attention([1, 7, 0, 64, 333, 95], 8, 8, 64), name="attention-tiny-packed"),
        # Llama-2-7B: one sequence of its whole context.
        dict(_attention([4096], 32, 32, 128), name="attention-7b"),
        # Llama-3-8B: documents of all lengths packed into 8192 tokens, four query heads to a key head.
        dict(_attention([2801, 17, 1209, 350, 64, 2444, 1, 906, 400], 32, 8, 128), name="attention-llama3-packed"),
        # One TP8 rank of Llama-2-70B in context parallelism: the last 2048 queries to 16384 gathered keys.
        dict(_attention([2048], 8, 1, 128, keys=[16384]), name="attention-70b-last-queries"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _parts(rng, total, count):
    """``count`` sizes that sum to ``total``, uneven, some of them zero."""
    cuts = sorted(rng.randrange(total + 1) for _ in range(count - 1))
    return [b - a for a, b in zip([0, *cuts], [*cuts, total])]


def _draw(rng):
    op = rng.choice(["norm", "experts", "attention"])
    dtype, train = rng.choice(["bf16", "bf16", "bf16", "fp16"]), rng.random() < 0.8
    if op == "norm":
        hidden = rng.choice([128, 512, 1000, 1024, 2048, 4096, 5120, 8192, _log_uniform(rng, 1, 8192), 8 * _log_uniform(rng, 4, 1024)])
        return _norm(_log_uniform(rng, 1, 8192), hidden, dtype, rng.choice([dtype, dtype, "fp32"]), rng.random() < 0.5,
                     rng.choice(["none", "none", "channel", "token"]), rng.choice([1.0, 1.0, round(rng.uniform(0.2, 1.5), 2)]), train)
    if op == "experts":
        count = rng.choice([1, 2, 2, 4, 8, 8, 16, 64])
        n_in, n_out = (rng.choice([128, 512, 1000, 1024, 1376, 4096, _log_uniform(rng, 8, 8192)]) for _ in range(2))
        if rng.random() < 0.3:
            n_in, n_out = n_in // 8 * 8 + 8, n_out // 8 * 8 + 8
        return _experts(_parts(rng, _log_uniform(rng, 1, 8192), count), n_in, n_out, dtype, rng.choice([0, 0, rng.randrange(100)]), train)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
    dim = rng.choice([32, 64, 64, 100, 128, 128, 128, rng.randrange(1, 129), 8 * rng.randrange(1, 17)])
    queries = _parts(rng, _log_uniform(rng, 1, 8192), rng.choice([1, 1, 2, 3, 5, 9, 20]))
    keys = queries
    if rng.random() < 0.25:  # the last queries of longer documents, and now and then fewer keys than queries
        keys = [n + _log_uniform(rng, 1, 4096) if rng.random() < 0.8 else n // 2 for n in queries]
    return _attention(queries, heads, kv_heads, dim, keys, dtype, rng.random() < 0.75, rng.choice([0, 0, rng.randrange(70)]), train)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


def _sizes(text):
    return [int(x) for x in text.split(",")]


def _bounds(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["train"]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    if case["op"] == "norm":
        t, h = case["tokens"], case["hidden"]
        # Deep in a model the stream is larger than what one block adds, and channels differ in size.
        channels = torch.randn(h, generator=gen, device="cuda").mul_(0.5).exp_()
        leaves = dict(residual=(torch.randn(t, h, generator=gen, device="cuda") * channels * 3).to(DTYPES[case["residual"]]),
                      branch=(torch.randn(t, h, generator=gen, device="cuda") * channels).to(dt),
                      weight=(1 + 0.2 * torch.randn(h, generator=gen, device="cuda")).to(dt))
        if case["branch_norm"]:
            leaves["branch_weight"] = (1 + 0.2 * torch.randn(h, generator=gen, device="cuda")).to(dt)
        if case["gate"] != "none":
            leaves["gate"] = normal(*((t, h) if case["gate"] == "token" else (h,)), scale=0.5)
        # Gradients as they reach a layer: small, and of the whole batch's size.
        grads = [normal(t, h, scale=1e-2, dtype=DTYPES[case["residual"]]), normal(t, h, scale=1e-2)]
    elif case["op"] == "experts":
        counts = _sizes(case["counts"])
        rows = sum(counts) + case["spare"]
        leaves = dict(x=normal(rows, case["n_in"]))
        for e in range(len(counts)):
            leaves["w%d" % e] = normal(case["n_out"], case["n_in"], scale=1 / math.sqrt(case["n_in"]))
        grads = [normal(rows, case["n_out"], scale=1e-2)]
    else:
        rows, key_rows = (sum(_sizes(case[k])) + case["spare"] for k in ("queries", "keys"))
        # Queries and keys as rotary embedding leaves them: scores that spread by about 2.
        leaves = dict(q=normal(rows, case["heads"], case["dim"], scale=1.5), k=normal(key_rows, case["kv_heads"], case["dim"], scale=1.5),
                      v=normal(key_rows, case["kv_heads"], case["dim"]))
        grads = [normal(rows, case["heads"], case["dim"], scale=1e-2)]
    if train:
        for x in leaves.values():
            x.requires_grad_()
    state = dict(case, leaves=leaves, grads=grads)
    if case["op"] == "experts":
        state["counts_on_device"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
    elif case["op"] == "attention":
        for k in ("queries", "keys"):
            state[k + "_from"] = torch.tensor(_bounds(_sizes(case[k])), dtype=torch.int32, device="cuda")
    return state


# ----- the plain forms -----


def _plain_norm(s):
    x = {k: v.detach().float() for k, v in s["leaves"].items()}
    dt, scale = DTYPES[s["dtype"]], s["scale"]
    branch, gate, weight = x["branch"], x.get("gate"), x["weight"]
    normed = branch
    if s["branch_norm"]:
        branch_rms = torch.rsqrt(branch.square().mean(1, keepdim=True) + EPS)
        unit = branch * branch_rms
        normed = unit * x["branch_weight"]
    stream = scale * x["residual"] + (normed if gate is None else gate * normed)
    rms = torch.rsqrt(stream.square().mean(1, keepdim=True) + EPS)
    hat = stream * rms
    out = [stream.to(s["leaves"]["residual"].dtype), (hat * weight).to(dt)]
    if not s["train"]:
        return out
    d_stream, d_out = (g.float() for g in s["grads"])
    d = d_out * weight
    d_stream = d_stream + rms * (d - hat * (d * hat).mean(1, keepdim=True))
    d_normed = d_stream if gate is None else d_stream * gate
    d_branch = d_normed
    if s["branch_norm"]:
        d = d_normed * x["branch_weight"]
        d_branch = branch_rms * (d - unit * (d * unit).mean(1, keepdim=True))
    out += [(scale * d_stream).to(s["leaves"]["residual"].dtype), d_branch.to(dt), (d_out * hat).sum(0).to(dt)]
    if s["branch_norm"]:
        out.append((d_normed * unit).sum(0).to(dt))
    if gate is not None:
        d_gate = d_stream * normed
        out.append((d_gate if s["gate"] == "token" else d_gate.sum(0)).to(dt))
    return out


def _plain_experts(s):
    x, dt = s["leaves"]["x"].detach(), DTYPES[s["dtype"]]
    dy = s["grads"][0]
    at = _bounds(_sizes(s["counts"]))
    y = torch.zeros(x.shape[0], s["n_out"], dtype=dt, device=x.device)
    dx, dws = torch.zeros_like(x), []
    for e, (lo, hi) in enumerate(zip(at, at[1:])):
        w = s["leaves"]["w%d" % e].detach().float() if hi > lo else None
        if hi > lo:
            y[lo:hi] = (x[lo:hi].float() @ w.t()).to(dt)
        if s["train"]:
            if hi > lo:
                dx[lo:hi] = (dy[lo:hi].float() @ w).to(dt)
            dws.append((dy[lo:hi].float().t() @ x[lo:hi].float()).to(dt))
    return [y, dx, *dws] if s["train"] else y


def _plain_attention(s):
    q, k, v = (s["leaves"][n].detach() for n in "qkv")
    dt, group = q.dtype, s["heads"] // s["kv_heads"]
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    q_at, k_at = _bounds(_sizes(s["queries"])), _bounds(_sizes(s["keys"]))
    scale = 1 / math.sqrt(s["dim"])
    for i in range(len(q_at) - 1):
        rows, cols = slice(q_at[i], q_at[i + 1]), slice(k_at[i], k_at[i + 1])
        n, m = q_at[i + 1] - q_at[i], k_at[i + 1] - k_at[i]
        if not n or not m:
            continue
        hidden = None
        if s["causal"]:  # the last query sees the last key
            hidden = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1)
        for g in range(s["kv_heads"]):
            heads = slice(g * group, (g + 1) * group)
            qh = q[rows, heads].float().transpose(0, 1).reshape(group * n, -1)
            kh, vh = k[cols, g].float(), v[cols, g].float()
            x = (qh @ kh.t().contiguous()).view(group, n, m) * scale
            if hidden is not None:
                x.masked_fill_(hidden, -math.inf)
            top = x.amax(2, keepdim=True)
            p = (x - torch.where(top == -math.inf, 0.0, top)).exp()
            total = p.sum(2, keepdim=True)
            p = (p / torch.where(total == 0, 1.0, total)).view(group * n, m)
            o = p @ vh
            out[rows, heads] = o.view(group, n, -1).transpose(0, 1).to(dt)
            if not s["train"]:
                continue
            do = s["grads"][0][rows, heads].float().transpose(0, 1).reshape(group * n, -1)
            dv[cols, g] = (p.t() @ do).to(dt)
            d = p * (do @ vh.t().contiguous() - (do * o).sum(1, keepdim=True)) * scale
            dq[rows, heads] = (d @ kh).view(group, n, -1).transpose(0, 1).to(dt)
            dk[cols, g] = (d.t() @ qh).to(dt)
    return [out, dq, dk, dv] if s["train"] else out


# ----- the framework's calls -----


def _framework(s):
    from elasticmegatron_amd import training

    x = s["leaves"]
    if s["op"] == "norm":
        outputs = training.residual_norm(x["residual"], x["branch"], x["weight"], branch_weight=x.get("branch_weight"), gate=x.get("gate"),
                                         residual_scale=s["scale"], eps=EPS)
        wanted = [x[k] for k in ("residual", "branch", "weight", "branch_weight", "gate") if k in x]
    elif s["op"] == "experts":
        wanted = list(x.values())
        outputs = [training.expert_linear(x["x"], wanted[1:], s["counts_on_device"])]
    else:
        keys = None if s["keys"] == s["queries"] else s["keys_from"]
        outputs = [training.attention(x["q"], x["k"], x["v"], offsets=s["queries_from"], key_offsets=keys, causal=s["causal"])]
        wanted = list(x.values())
    if not s["train"]:
        return list(outputs) if len(outputs) > 1 else outputs[0]
    return [*outputs, *torch.autograd.grad(outputs, wanted, s["grads"])]


def run(state):
    if own:
        return _framework(state)
    return {"norm": _plain_norm, "experts": _plain_experts, "attention": _plain_attention}[state["op"]](state)


# ----- what they cannot do without -----


def _pairs(case):
    """Pairs of a query and a key that it sees, of one head."""
    total = 0
    for n, m in zip(_sizes(case["queries"]), _sizes(case["keys"])):
        if case["causal"]:  # query i sees i + 1 + m - n keys, where that is positive
            first = max(0, n - m)
            total += (n - first) * (max(0, m - n) + 1 + m) // 2
        else:
            total += n * m
    return total


def work(case):
    if case["op"] == "norm":
        n, h = case["tokens"] * case["hidden"], case["hidden"]
        r = 4 if case["residual"] == "fp32" else 2
        gate = {"none": 0, "channel": 2 * h, "token": 2 * n}[case["gate"]]
        weights = 2 * h * (2 if case["branch_norm"] else 1)
        moved, flops = n * (2 * r + 4) + gate + weights, n * 8
        if case["train"]:
            moved, flops = moved + n * (2 * r + 4) + gate + weights, n * 30
        return {"bytes": moved, "flops": flops}
    if case["op"] == "experts":
        counts = _sizes(case["counts"])
        rows, used = sum(counts), sum(c > 0 for c in counts)
        weight = case["n_in"] * case["n_out"]
        moved = 2 * (rows * case["n_in"] + used * weight + (rows + case["spare"]) * case["n_out"])
        if case["train"]:  # the other gradients' sides are read and written too, every expert's among them
            moved += 2 * (rows * case["n_out"] + (rows + case["spare"]) * case["n_in"] + len(counts) * weight)
        return {"bytes": moved, "flops": (6 if case["train"] else 2) * rows * weight}
    rows, keys = (sum(_sizes(case[k])) for k in ("queries", "keys"))
    one, both = 2 * case["heads"] * case["dim"] * rows, 4 * case["kv_heads"] * case["dim"] * keys
    moved = 2 * one + both
    if case["train"]:
        moved += 2 * one + both
    return {"bytes": moved, "flops": (14 if case["train"] else 4) * _pairs(case) * case["heads"] * case["dim"]}


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 1e15


# ----- 64 bits, from the definitions -----


def _rms(x, weight):
    return x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight


def _exact_norm(case, s):
    x = {k: v.detach().double().requires_grad_(case["train"]) for k, v in s["leaves"].items()}
    branch = _rms(x["branch"], x["branch_weight"]) if case["branch_norm"] else x["branch"]
    stream = x["residual"] * case["scale"] + branch * x.get("gate", 1.0)
    outputs = [stream, _rms(stream, x["weight"])]
    if not case["train"]:
        return outputs
    wanted = [x[k] for k in ("residual", "branch", "weight", "branch_weight", "gate") if k in x]
    return [*(o.detach() for o in outputs), *torch.autograd.grad(outputs, wanted, [g.double() for g in s["grads"]])]


def _exact_experts(case, s):
    tokens, weights = s["leaves"]["x"].detach().double(), [v.detach() for k, v in s["leaves"].items() if k != "x"]
    dy = s["grads"][0].double()
    counts = _sizes(case["counts"])
    y, dx, dws = [], [], []
    parts = torch.split(tokens, [*counts, case["spare"]])
    grads = torch.split(dy, [*counts, case["spare"]])
    for a, d, w in zip(parts, grads, weights):
        w = w.double()
        y.append(torch.mm(a, w.t()))
        if case["train"]:
            dx.append(torch.mm(d, w))
            dws.append(torch.mm(d.t(), a))
    y = torch.cat([*y, torch.zeros_like(grads[-1])])
    return [y, torch.cat([*dx, torch.zeros_like(parts[-1])]), *dws] if case["train"] else y


def _exact_attention(case, s):
    q, k, v = (s["leaves"][n].detach().double() for n in "qkv")
    do = s["grads"][0].double()
    share = case["heads"] // case["kv_heads"]
    out, gq, gk, gv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    lo = at = 0
    for n, m in zip(_sizes(case["queries"]), _sizes(case["keys"])):
        see = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if case["causal"]:
            i, j = torch.arange(n, device=q.device)[:, None], torch.arange(m, device=q.device)[None]
            see = j - m <= i - n
        full = see.any(1) if m else see.new_zeros(n)
        for h in range(case["heads"] if n and m else 0):
            a, b, c = q[lo:lo + n, h], k[at:at + m, h // share], v[at:at + m, h // share]
            score = torch.mm(a, b.t()) / math.sqrt(case["dim"])
            p = torch.softmax(score.masked_fill(~see, -math.inf), 1)
            p[~full] = 0
            o = torch.mm(p, c)
            out[lo:lo + n, h] = o
            if case["train"]:
                d = do[lo:lo + n, h]
                gv[at:at + m, h // share] += torch.mm(p.t(), d)
                ds = p * (torch.mm(d, c.t()) - (d * o).sum(1)[:, None]) / math.sqrt(case["dim"])
                gq[lo:lo + n, h] = torch.mm(ds, b)
                gk[at:at + m, h // share] += torch.mm(ds.t(), a)
        lo, at = lo + n, at + m
    return [out, gq, gk, gv] if case["train"] else out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "experts": _exact_experts, "attention": _exact_attention}[case["op"]](case, s)
