"""Cases for the operators around a linear-time language model: decay attention (linear attention with a decay for
each head; whole sequences, training and single tokens), the embedding lookup with its gradient, and token sampling.

`run` is one call as a user's program makes it: with `own` the framework's operators, without it the same results from
elementary torch operations in 32 bits."""

import math

import torch

own = False

VOCAB = 50304  # the vocabulary of the 60M and 125M models


def listed():
    return [
        # One decode step of 64 sequences: the rows of the current tokens, scaled, in the residual's type.
        dict(name="lookup of a decode step", op="lookup", tokens=64, vocab=VOCAB, dim=512, weight="f32", out="bf16"),
        # The 60M model's training step (32 x 1024 tokens, width 512): lookup and gradient of the float32 table.
        dict(name="embedding of a 60M step", op="embed", tokens=32768, vocab=VOCAB, dim=512, weight="f32", out="bf16"),
        # The 125M model's step (64 x 1024 tokens, width 768).
        dict(name="embedding of a 125M step", op="embed", tokens=65536, vocab=VOCAB, dim=768, weight="f32", out="bf16"),
        # One sequence generating: latency.
        dict(name="sample one sequence", op="sample", rows=1, vocab=VOCAB, dtype="f32", mix="usual"),
        # 64 sequences of one decode step, each row with its own settings (greedy and unfiltered rows among them).
        dict(name="sample 64 mixed rows", op="sample", rows=64, vocab=VOCAB, dtype="f32", mix="mixed"),
        # A large serving batch over a large vocabulary, bfloat16 logits.
        dict(name="sample 512 wide rows", op="sample", rows=512, vocab=131072, dtype="bf16", mix="nucleus"),
        # One token of one sequence: key 64, value 128, 8 heads (the memory mixer's layout at width 512).
        dict(name="step of one sequence", op="step", batch=1, heads=8, kv=8, dk=64, dv=128, dtype="bf16"),
        # One token of a decode batch with square heads.
        dict(name="step of 64 sequences", op="step", batch=64, heads=16, kv=16, dk=128, dv=128, dtype="bf16"),
        # A long prompt of one sequence: few rows, a long time axis.
        dict(name="long prompt", op="prompt", batch=1, time=32768, heads=8, kv=8, dk=128, dv=128, dtype="bf16", ragged=False),
        # Prompts of different lengths continuing earlier states, odd head sizes, shared key/value heads, one projection.
        dict(name="ragged prompts", op="prompt", batch=5, time=777, heads=6, kv=2, dk=80, dv=96, dtype="bf16", ragged=True),
        # The mixer in the 60M training step: 32 x 1024 tokens, 8 heads, key 64, value 128.
        dict(name="training step", op="train", batch=32, time=1024, heads=8, kv=8, dk=64, dv=128, dtype="bf16"),
        # float32 operands, odd sizes, carried state with its gradient.
        dict(name="float32 training, odd sizes", op="train", batch=3, time=333, heads=4, kv=4, dk=40, dv=72, dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("lookup", "embed", "sample", "step", "prompt", "train", "sample", "prompt", "train"))
    if op in ("lookup", "embed"):
        tokens = _log_int(rng, 1, 4096) if op == "lookup" else _log_int(rng, 100, 65536)
        return dict(op=op, tokens=tokens, vocab=_log_int(rng, 500, 60000), dim=8 * rng.randint(8, 96),
                    weight=rng.choice(("f32", "f32", "bf16")), out=rng.choice(("bf16", "bf16", "f32")))
    if op == "sample":
        return dict(op=op, rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 300, 131072), dtype=rng.choice(("f32", "bf16")),
                    mix=rng.choice(("usual", "mixed", "nucleus")))
    kv = rng.choice((1, 2, 3, 4, 8))
    dims = dict(kv=kv, heads=kv * rng.choice((1, 1, 1, 2, 3)), dk=8 * rng.randint(2, 16), dv=8 * rng.randint(2, 16))
    if op == "step":
        return dict(op=op, batch=_log_int(rng, 1, 32), dtype=rng.choice(("bf16", "f32")), **dims)
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    time = _log_int(rng, 1, 4096 if dtype == "bf16" else 1024)
    batch = max(1, min(16, _log_int(rng, 1, 16384) // time))
    if op == "prompt":
        return dict(op=op, batch=batch, time=time, dtype=dtype, ragged=rng.random() < 0.5, **dims)
    return dict(op=op, batch=batch, time=time, dtype=dtype, **dims)


def _type(name):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


# ------------------------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------------------------
def _decays(heads):
    """Half lives from about 20 to about 2800 tokens, spread over the heads."""
    rate = 2.0 ** -torch.linspace(5.0, 12.0, heads, dtype=torch.float64)
    return torch.log1p(-rate).float().cuda()


def _settings(rows, mix, g):
    if mix == "usual":      # the same settings for every row, as plain numbers
        return dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.0)
    if mix == "nucleus":
        return dict(temperature=1.0, top_k=0, top_p=0.9, min_p=0.0)
    pick = lambda values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]  # noqa: E731
    return dict(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3]), top_k=pick([0, 0, 1, 20, 50, 1000]).to(torch.int32),
                top_p=pick([1.0, 1.0, 0.95, 0.9, 0.5]), min_p=pick([0.0, 0.0, 0.0, 0.02, 0.1]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case=case)
    if op in ("lookup", "embed"):
        n, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        # Token frequencies fall with the rank as in text (about 1 / rank); ids in random order; a few padded places.
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        rank = torch.clamp((torch.exp(u * math.log(vocab + 1.0)) - 1.0).long(), 0, vocab - 1)
        s["tokens"] = torch.randperm(vocab, generator=g, device="cuda")[rank]
        s["tokens"][torch.rand(n, generator=g, device="cuda") < 0.01] = -1
        s["weight"] = (0.02 * torch.randn(vocab, dim, generator=g, device="cuda")).to(_type(case["weight"]))
        s["weight"].requires_grad_(op == "embed")
        s["scale"] = math.sqrt(dim)
        s["out"] = _type(case["out"])
        if op == "embed":
            s["grad"] = torch.randn(n, dim, generator=g, device="cuda").to(s["out"])
        return s
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # A few likely tokens over a broad tail, as a trained head gives them; some rows sharper than others.
        logits = 2.2 * torch.randn(rows, vocab, generator=g, device="cuda")
        logits += 1.5 * torch.rand(rows, 1, generator=g, device="cuda") * torch.randn(rows, vocab, generator=g, device="cuda").abs()
        if case["mix"] == "mixed":  # a grammar's mask: part of the vocabulary ruled out
            logits[:, torch.rand(vocab, generator=g, device="cuda") < 0.3] = -torch.inf
        s["logits"] = logits.to(_type(case["dtype"]))
        s["uniform"] = torch.rand(rows, generator=g, device="cuda")
        s["settings"] = _settings(rows, case["mix"], g)
        return s
    b, h, kv, dk, dv, dtype = (case[n] for n in ("batch", "heads", "kv", "dk", "dv", "dtype"))
    dtype = _type(dtype)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s["log_decay"] = _decays(h)
    s["scale"] = dk ** -0.5
    if op == "step":
        s["q"], s["k"], s["v"] = (rand(b, n, d).to(dtype) for n, d in ((h, dk), (kv, dk), (kv, dv)))
        s["state"] = 3.0 * rand(b, h, dk, dv)
        return s
    t = case["time"]
    if op == "prompt":  # slices of one projection, as a model has them
        proj = rand(b, t, h * dk + kv * dk + kv * dv).to(dtype)
        q, k, v = proj.split([h * dk, kv * dk, kv * dv], dim=-1)
        s["q"], s["k"], s["v"] = q.view(b, t, h, dk), k.view(b, t, kv, dk), v.view(b, t, kv, dv)
        s["initial"] = s["lengths"] = None
        if case["ragged"]:
            s["lengths"] = torch.randint(0, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            s["lengths"][0] = t
            s["initial"] = rand(b, h, dk, dv)
        return s
    s["q"], s["k"], s["v"] = (rand(b, t, n, d).to(dtype).requires_grad_(True) for n, d in ((h, dk), (kv, dk), (kv, dv)))
    s["initial"] = rand(b, h, dk, dv).requires_grad_(True)
    s["d_output"], s["d_state"] = rand(b, t, h, dv).to(dtype), rand(b, h, dk, dv)
    return s


# ------------------------------------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------------------------------------
def _plain_attention(q, k, v, log_decay, scale, initial, lengths):
    """Chunks of 64 tokens: products inside a chunk, and a decayed sum of the chunks' states."""
    b, t, h, dk = q.shape
    dv, dtype, c = v.shape[-1], q.dtype, 64
    group = h // k.shape[2]
    q, k, v = q.float(), k.float().repeat_interleave(group, 2), v.float().repeat_interleave(group, 2)
    steps = torch.arange(t, device=q.device)
    if lengths is None:
        left = (t - 1 - steps).expand(b, t)
    else:
        left = lengths[:, None] - 1 - steps
        inside = (left >= 0)[:, :, None, None]
        q, k, v = (torch.where(inside, x, 0.0) for x in (q, k, v))
    length = torch.full((b,), t, device=q.device) if lengths is None else lengths
    g = log_decay
    weight = torch.exp(g * left.clamp(min=0)[..., None])[..., None]                                  # [b, t, h, 1]
    final = torch.matmul((k * weight).permute(0, 2, 3, 1), v.transpose(1, 2))
    if initial is not None:
        final = final + torch.exp(g * length[:, None])[..., None, None] * initial
    n = -(-t // c)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * c - t)).view(b, n, c, h, -1).permute(0, 3, 1, 2, 4) for x in (q, k, v))
    i = torch.arange(c, device=q.device)
    gap = i[:, None] - i
    inner = torch.where(gap >= 0, torch.exp(g[:, None, None] * gap.clamp(min=0)), 0.0)               # [h, c, c]
    out = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * inner[:, None], v)
    end = torch.exp(g[:, None] * (c - 1 - i))                                                        # [h, c]
    local = torch.matmul((k * end[:, None, :, None]).transpose(-1, -2), v)                           # [b, h, n, dk, dv]
    m = torch.arange(n, device=q.device)
    hops = m[:, None] - 1 - m
    carry = torch.where(hops >= 0, torch.exp(g[:, None, None] * c * hops.clamp(min=0)), 0.0)         # [h, n, n]
    start = torch.matmul(carry, local.reshape(b, h, n, dk * dv)).view(b, h, n, dk, dv)
    if initial is not None:
        start = start + torch.exp(g[:, None] * c * m)[..., None, None] * initial[:, :, None]
    out = out + torch.matmul(q * torch.exp(g[:, None] * (i + 1))[:, None, :, None], start)
    return (scale * out).permute(0, 2, 3, 1, 4).reshape(b, n * c, h, dv)[:, :t].to(dtype), final


def _plain_step(state, q, k, v, log_decay, scale):
    group = q.shape[1] // k.shape[1]
    kf, vf = k.float().repeat_interleave(group, 1), v.float().repeat_interleave(group, 1)
    state = torch.exp(log_decay)[:, None, None] * state + kf[..., :, None] * vf[..., None, :]
    return (scale * torch.matmul(q.float()[..., None, :], state)[..., 0, :]).to(q.dtype), state


def _plain_sample(logits, uniform, temperature, top_k, top_p, min_p):
    rows, vocab = logits.shape
    row = lambda x, dtype: torch.as_tensor(x, device=logits.device).to(dtype).expand(rows)[:, None]  # noqa: E731
    temperature, top_k, top_p, min_p = row(temperature, torch.float32), row(top_k, torch.int64), row(top_p, torch.float32), row(min_p, torch.float32)
    x = logits.float()
    x = torch.where(torch.isnan(x), -torch.inf, x)
    top = x.amax(-1, keepdim=True)
    greedy = ~(temperature > 0)
    z = torch.where(x == top, 0.0, (top - x) * torch.where(greedy, 1.0, 1.0 / temperature))
    e = torch.exp(-z)
    mass = (e * 2.0 ** 35).to(torch.int64)
    order = torch.sort(z, dim=-1, stable=True).indices
    sorted_mass = mass.gather(-1, order)
    rank = torch.arange(vocab, device=x.device)
    limit_k = torch.where(greedy, 1, torch.where(top_k > 0, top_k, vocab))
    keep = rank < limit_k
    running = torch.cumsum(sorted_mass * keep, -1)
    limit_p = torch.ceil(top_p.double() * running[:, -1:].double()).to(torch.int64)
    keep = keep & ((running - sorted_mass < limit_p) | (top_p >= 1) | (rank == 0)) & ((e.gather(-1, order) >= min_p) | (rank == 0))
    kept = torch.zeros_like(mass).scatter(-1, order, sorted_mass * keep)
    running = torch.cumsum(kept, -1)
    total = running[:, -1:]
    target = torch.minimum((uniform[:, None].double() * total.double()).floor().to(torch.int64).clamp(min=0), total - 1)
    token = (running <= target).sum(-1)
    log_prob = -z.gather(-1, token[:, None])[:, 0] - torch.log((total[:, 0].double() * 2.0 ** -35).float())
    empty = top[:, 0] == -torch.inf  # nothing left by the mask
    return torch.where(empty, -1, token), torch.where(empty, -torch.inf, log_prob)


def _plain_lookup(tokens, weight, scale, out):
    inside = (tokens >= 0) & (tokens < weight.shape[0])
    rows = weight[torch.where(inside, tokens, 0)].float() * scale
    return torch.where(inside[:, None], rows, 0.0).to(out)


def _plain_lookup_grad(tokens, weight, scale, grad):
    vocab = weight.shape[0]
    inside = (tokens >= 0) & (tokens < vocab)
    table = torch.zeros(vocab + 1, weight.shape[1], device=weight.device)
    table.index_add_(0, torch.where(inside, tokens, vocab), grad.float())
    return (scale * table[:vocab]).to(weight.dtype)


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        import mamba4_b200 as m4

        if op == "lookup":
            return m4.embedding_lookup(s["tokens"], s["weight"], scale=s["scale"], dtype=s["out"])
        if op == "embed":
            rows = m4.embedding_lookup(s["tokens"], s["weight"], scale=s["scale"], dtype=s["out"])
            return rows.detach(), torch.autograd.grad(rows, s["weight"], s["grad"])[0]
        if op == "sample":
            got = m4.sample_tokens(s["logits"], s["uniform"], **s["settings"])
            return got.tokens, got.log_prob
        if op == "step":
            got = m4.decay_attention_step(s["state"], s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"])
            return got.output, got.state
        got = m4.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], initial=s["initial"], lengths=s.get("lengths"))
        out, final = got.output, got.state
    elif op == "lookup":
        return _plain_lookup(s["tokens"], s["weight"], s["scale"], s["out"])
    elif op == "embed":
        weight = s["weight"].detach()
        return _plain_lookup(s["tokens"], weight, s["scale"], s["out"]), _plain_lookup_grad(s["tokens"], weight, s["scale"], s["grad"])
    elif op == "sample":
        return _plain_sample(s["logits"], s["uniform"], **s["settings"])
    elif op == "step":
        return _plain_step(s["state"], s["q"], s["k"], s["v"], s["log_decay"], s["scale"])
    else:
        out, final = _plain_attention(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["initial"], s.get("lengths"))
    if op == "prompt":
        return out, final
    leaves = (s["q"], s["k"], s["v"], s["initial"])
    return (out.detach(), final.detach()) + torch.autograd.grad((out, final), leaves, (s["d_output"], s["d_state"]))


# ------------------------------------------------------------------------------------------------------------------
# Work and exact values
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2}
    if op in ("lookup", "embed"):
        n, vocab, dim, w, o = case["tokens"], case["vocab"], case["dim"], size[case["weight"]], size[case["out"]]
        seen = vocab * (1 - math.exp(-n * 1.0 / vocab)) if op == "lookup" else min(n, vocab)
        lookup = dict(bytes=8 * n + min(n, seen) * dim * w + n * dim * o, flops=n * dim)
        if op == "lookup":
            return lookup
        return dict(bytes=lookup["bytes"] + n * dim * o + vocab * dim * w, flops=2 * n * dim + vocab * dim)
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * size[case["dtype"]] + case["rows"] * 36, flops=6 * n)
    b, h, kv, dk, dv, w = case["batch"], case["heads"], case["kv"], case["dk"], case["dv"], size[case["dtype"]]
    per_token = b * w * (h * dk + kv * dk + kv * dv + h * dv)
    states = 4 * b * h * dk * dv
    if op == "step":
        return dict(bytes=per_token + 2 * states, flops=5 * b * h * dk * dv)
    t = case["time"]
    if op == "prompt":
        return dict(bytes=t * per_token + states * (2 if case["ragged"] else 1), flops=4 * b * t * h * dk * dv)
    return dict(bytes=t * 2 * per_token + 4 * states, flops=14 * b * t * h * dk * dv)


def exact(case, seed):
    def attention(s):
        """The whole attention matrix of each row and head, in blocks of query rows."""
        q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
        b, t, h, dk = q.shape
        kv, dv = k.shape[2], v.shape[-1]
        group = h // kv
        lengths = s["lengths"].tolist() if s.get("lengths") is not None else [t] * b
        initial = torch.zeros(b, h, dk, dv, dtype=torch.float64, device=q.device) if s["initial"] is None else s["initial"].detach().double()
        out, final = torch.zeros(b, t, h, dv, dtype=torch.float64, device=q.device), torch.zeros_like(initial)
        train = "d_output" in s
        if train:
            d_out, d_fin = s["d_output"].double(), s["d_state"].double()
            dq, dk_, dv_, d_init = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(initial)
        gs, scale = s["log_decay"].double().tolist(), s["scale"]
        for r in range(b):
            n = lengths[r]
            age = torch.arange(n, dtype=torch.float64, device=q.device)
            for a in range(h):
                g, c = gs[a], a // group
                qa, ka, va, s0 = q[r, :n, a], k[r, :n, c], v[r, :n, c], initial[r, a]
                to_end, from_start = torch.exp(g * (n - 1 - age))[:, None], torch.exp(g * (age + 1))[:, None]
                final[r, a] = (ka * to_end).T @ va + math.exp(g * n) * s0
                if train:
                    df = d_fin[r, a]
                    dk_[r, :n, c] += to_end * (va @ df.T)
                    dv_[r, :n, c] += to_end * (ka @ df)
                    do = d_out[r, :n, a]
                    dq[r, :n, a] += scale * from_start * (do @ s0.T)
                    d_init[r, a] = math.exp(g * n) * df + scale * (qa * from_start).T @ do
                out[r, :n, a] = scale * from_start * (qa @ s0)
                for x in range(0, n, 2048):
                    y = min(n, x + 2048)
                    gap = age[x:y, None] - age[None, :y]
                    w = torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), 0.0) * scale
                    p = (qa[x:y] @ ka[:y].T) * w
                    out[r, x:y, a] += p @ va[:y]
                    if train:
                        dp = (do[x:y] @ va[:y].T) * w
                        dq[r, x:y, a] += dp @ ka[:y]
                        dk_[r, :y, c] += dp.T @ qa[x:y]
                        dv_[r, :y, c] += p.T @ do[x:y]
        return (out, final, dq, dk_, dv_, d_init) if train else (out, final)

    s = prepare(case, seed)
    op = case["op"]
    if op in ("lookup", "embed"):
        tokens, weight = s["tokens"], s["weight"].detach().double()
        inside = (tokens >= 0) & (tokens < case["vocab"])
        rows = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device=tokens.device)
        rows[inside] = weight[tokens[inside]] * s["scale"]
        if op == "lookup":
            return rows
        table = torch.zeros_like(weight)
        table.index_put_((tokens[inside],), s["grad"][inside].double(), accumulate=True)
        return rows, table * s["scale"]
    if op == "sample":
        x = s["logits"].double().cpu()
        u = s["uniform"].double().tolist()
        settings = {n: (v.tolist() if torch.is_tensor(v) else [v] * len(u)) for n, v in s["settings"].items()}
        log_prob = torch.zeros(len(u), dtype=torch.float64)
        for r in range(len(u)):
            if x[r].max() == -torch.inf:
                log_prob[r] = -torch.inf
                continue
            hot = settings["temperature"][r] > 0
            p = torch.softmax(x[r] / (settings["temperature"][r] if hot else 1.0), 0)
            sorted_p, order = torch.sort(p, descending=True, stable=True)
            count = (settings["top_k"][r] or case["vocab"]) if hot else 1
            sorted_p[count:] = 0
            before = torch.cumsum(sorted_p, 0) - sorted_p
            if settings["top_p"][r] < 1:
                sorted_p = torch.where((before < settings["top_p"][r] * sorted_p.sum()) | (before == 0), sorted_p, 0.0)
            sorted_p = torch.where(sorted_p >= settings["min_p"][r] * sorted_p[0], sorted_p, 0.0)
            kept = torch.zeros_like(p).scatter(0, order, sorted_p / sorted_p.sum())
            running = torch.cumsum(kept, 0)
            token = min(int((running <= u[r] * running[-1]).sum()), case["vocab"] - 1)
            log_prob[r] = torch.log(kept[token])
        return None, log_prob
    if op == "step":
        group = case["heads"] // case["kv"]
        head = torch.arange(case["heads"], device="cuda") // group
        state = torch.exp(s["log_decay"].double())[:, None, None] * s["state"].double()
        state = state + torch.einsum("bhx,bhy->bhxy", s["k"].double()[:, head], s["v"].double()[:, head])
        return s["scale"] * torch.einsum("bhx,bhxy->bhy", s["q"].double(), state), state
    return attention(s)
