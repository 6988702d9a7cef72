"""What the operators of an 8-bit decoding step are measured on: matrix
products in 8-bit integers with a scale for each token and channel (plain,
and as a SwiGLU), and drawing tokens from logits by given uniform numbers.

``run`` computes each operator in elementary torch operations (``own`` false)
or through ``soraku_tts_b200.kernels`` (``own`` true); ``exact`` restates the
definition in 64 bits.

A row y of activations (x, or x times a norm's weight, in FP32) becomes codes
round(y / s), s = max |y| / 127, with the quotient rounded to FP32 first; its
scale is s, with a norm divided by the row's root mean square.  Sums of products
of codes are exact.  Tokens are drawn in the order of the logits, the largest
first and equal ones by index: the first whose running sum of weights passes u
times their sum.
"""

import math

import torch

own = False

EPS = 1e-6


def listed():
    return [
        # one frame's QKV projection of one utterance's two guidance rows (latency counts)
        _product("linear_frame", "linear", 2, 1024, 4096, norm=True),
        # all 16 classifiers of a frame's codebooks for the two rows: bound by the weights' bytes
        _product("linear_classifiers", "linear", 2, 1024, 16 * 2051, norm=True, bias=True),
        # the output projection of a small batch's rows, onto the residual stream
        _product("linear_out_batch", "linear", 16, 2048, 1024, residual=True),
        # the QKV projection of a full batch's rows
        _product("linear_batch", "linear", 128, 1024, 4096, norm=True),
        # the QKV projection of eight whole prompts
        _product("linear_prompts", "linear", 6541, 1024, 4096, norm=True),
        # a wide layer over a long document, 16-bit activations
        _product("linear_wide_bf16", "linear", 4096, 4096, 4096, dtype="bfloat16"),
        # the depth head's gate and up products for the two rows (latency counts)
        _product("swiglu_frame", "swiglu", 2, 1024, 2048, norm=True),
        # the same for a batch of odd width
        _product("swiglu_batch", "swiglu", 77, 1024, 2048, norm=True),
        # a wide MLP over several prompts, 16-bit activations
        _product("swiglu_prompts_bf16", "swiglu", 5003, 2048, 4096, norm=True, dtype="bfloat16"),
        # one codebook's code for each of 64 running utterances
        _sample("sample_codes", 64, 2051, temperature=0.9, top_k=50, top_p=0.95, min_p=0.05),
        # one text token of one utterance (latency counts): no top-k, the whole vocabulary has weight
        _sample("sample_text", 1, 151936, temperature=1.0, top_p=0.95, min_p=0.01),
        # a full batch of text tokens, every row with settings of its own
        _sample("sample_text_batch", 128, 151936, temperature=0.8, top_k=1000, top_p=0.9, min_p=0.02, per_row=True),
    ]


def _product(name, op, tokens, inner, outer, norm=False, bias=False, residual=False, dtype="float32"):
    return {"name": name, "op": op, "tokens": tokens, "inner": inner, "outer": outer, "norm": norm, "bias": bias,
            "residual": residual, "dtype": dtype}


def _sample(name, rows, vocab, temperature, top_k=0, top_p=1.0, min_p=0.0, per_row=False, dtype="float32"):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "per_row": per_row, "dtype": dtype}


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "swiglu", "sample"])
    dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
    if op == "sample":
        while True:
            rows, vocab = _spread(rng, 1, 512), _spread(rng, 100, 151936)
            if rows * vocab <= 128 * 151936:
                break
        case = _sample("", rows, vocab, temperature=round(rng.uniform(0.3, 1.5), 3),
                       top_k=rng.choice([0, 0, 20, 50, _spread(rng, 1, vocab)]), top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]),
                       min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]), per_row=rng.random() < 0.3, dtype=dtype)
    else:
        while True:
            tokens, inner, outer = _spread(rng, 1, 8192), _spread(rng, 32, 8192), _spread(rng, 16, 16 * 2051)
            if rng.random() < 0.6:
                inner, outer = -(-inner // 64) * 64, -(-outer // 64) * 64
            if tokens * inner * outer * (2 if op == "swiglu" else 1) <= 4096 ** 3 and tokens * outer <= 6541 * 4096:
                break
        case = _product("", op, tokens, inner, outer, norm=rng.random() < 0.5, bias=op == "linear" and rng.random() < 0.3,
                        residual=op == "linear" and rng.random() < 0.4, dtype=dtype)
    del case["name"]
    return case


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # rows between sharp and flat, one logit in a hundred masked (never a row's first, so that none is empty)
        logits = normal(rows, vocab) * (1.5 + 2.5 * torch.rand(rows, 1, generator=g, device=dev))
        masked = torch.rand(rows, vocab, generator=g, device=dev) < 0.01
        masked[:, 0] = False
        s = {"op": "sample", "logits": logits.masked_fill_(masked, -math.inf).to(dtype),
             "uniform": torch.rand(rows, generator=g, device=dev)}
        names = ("temperature", "top_k", "top_p", "min_p")
        if case["per_row"]:
            # rows' own settings, around the case's
            f = 0.75 + 0.5 * torch.rand(4, rows, generator=g, device=dev)
            s["temperature"] = case["temperature"] * f[0]
            s["top_k"] = (case["top_k"] * f[1]).to(torch.int32)
            s["top_p"] = (case["top_p"] * f[2]).clamp_(max=1.0)
            s["min_p"] = case["min_p"] * f[3]
        else:
            s.update({n: case[n] for n in names})
        return s
    tokens, inner, outer = case["tokens"], case["inner"], case["outer"]
    # activations with a few channels that stand out, as those of language models do
    x = normal(tokens, inner) * torch.where(torch.rand(inner, generator=g, device=dev) < 0.01, 12.0, 1.0)
    s = {"op": case["op"], "x": x.to(dtype), "norm": 1 + 0.2 * normal(inner) if case["norm"] else None,
         "bias": normal(outer) if case["bias"] else None, "residual": normal(tokens, outer).to(dtype) if case["residual"] else None}

    def weight():
        # codes and scales, laid out once: rows begin on 16 bytes
        codes, scale = _codes(normal(outer, inner) * 0.02)
        q = torch.zeros(outer, -(-inner // 16) * 16, dtype=torch.int8, device=dev)[:, :inner]
        return q.copy_(codes), scale

    s["w"] = [weight() for _ in range(2 if case["op"] == "swiglu" else 1)]
    return s


def run(state):
    if state["op"] == "sample":
        return _run_sample(state)
    if own:
        from soraku_tts_b200 import kernels

        if state["op"] == "linear":
            return kernels.int8_linear(state["x"], state["w"][0], norm_weight=state["norm"], eps=EPS, bias=state["bias"],
                                       residual=state["residual"])
        return kernels.int8_swiglu(state["x"], state["w"][0], state["w"][1], norm_weight=state["norm"], eps=EPS)
    return _plain_product(state)


def _codes(y):
    s = torch.clamp(y.abs().amax(-1) / 127, min=2.0 ** -126)
    return torch.round(y / s[:, None]), s


def _plain_product(s):
    x = s["x"].float()
    codes, scale = _codes(x if s["norm"] is None else x * s["norm"])
    if s["norm"] is not None:
        scale = scale * torch.rsqrt((x * x).mean(-1) + EPS)
    # sums of products of codes pass 2^24: 64 bits hold them exactly
    y = [(codes.double() @ w.double().T).float() * scale[:, None] * ws for w, ws in s["w"]]
    if s["op"] == "swiglu":
        return (y[0] / (1 + torch.exp(-y[0])) * y[1]).to(s["x"].dtype)
    y = y[0]
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _run_sample(s):
    settings = {n: s[n] for n in ("temperature", "top_k", "top_p", "min_p")}
    if own:
        from soraku_tts_b200 import kernels

        tokens, logprob = kernels.sample_tokens(s["logits"], s["uniform"], **settings)
    else:
        tokens, logprob = _plain_sample(s["logits"], s["uniform"], **settings)
    return {"tokens": tokens, "logprob": logprob}


def _column(x, dtype, like):
    x = x if isinstance(x, torch.Tensor) else torch.full(like.shape, x, dtype=dtype, device=like.device)
    return (x.double() if dtype is torch.float32 else x.long())[:, None]


def _plain_sample(logits, uniform, temperature, top_k, top_p, min_p):
    # 64 bits: a draw goes by running sums over up to 151,936 weights, and so does the border of top-p
    T, p, m = (_column(x, torch.float32, uniform) for x in (temperature, top_p, min_p))
    k = _column(top_k, torch.int32, uniform)
    value, index = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    place = torch.arange(logits.shape[1], device=logits.device)
    gap = (value - value[:, :1]) / T
    weight = torch.exp(gap)
    total = torch.cumsum(torch.where((k <= 0) | (place < k), weight, 0.0), 1)
    before = torch.cat([torch.zeros_like(T), total[:, :-1]], 1)
    kept = ((k <= 0) | (place < k)) & ((p >= 1) | (before < p * total[:, -1:])) & (weight >= m)
    last = kept.sum(1, keepdim=True) - 1
    mass = torch.gather(total, 1, last)
    passed = kept & (total <= uniform.double()[:, None] * mass)
    drawn = torch.minimum(passed.sum(1, keepdim=True), last)
    logprob = torch.gather(gap, 1, drawn) - torch.log(mass)
    return torch.gather(index, 1, drawn)[:, 0], logprob[:, 0].float()


def work(case):
    size = getattr(torch, case["dtype"]).itemsize
    if case["op"] == "sample":
        # logits in; a difference, a product and an exponential each
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (16 + (16 if case["per_row"] else 0)), "flops": 3 * n}
    t, k, n = case["tokens"], case["inner"], case["outer"]
    parts = 2 if case["op"] == "swiglu" else 1
    nbytes = t * k * size + parts * n * (k + 4) + t * n * size * (2 if case["residual"] else 1)
    return {"bytes": nbytes + (4 * k if case["norm"] else 0) + (4 * n if case["bias"] else 0), "flops": 2 * t * k * n * parts}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    x = s["x"].double()
    # products and quotients of FP32 values are rounded to FP32 by definition: a code is what it is
    y = x if s["norm"] is None else (x * s["norm"].double()).float().double()
    step = torch.clamp((y.abs().max(1, keepdim=True).values / 127).float().double(), min=2.0 ** -126)
    rows = torch.round((y / step).float().double()) * step
    if s["norm"] is not None:
        rows = rows / torch.sqrt((x ** 2).sum(1, keepdim=True) / x.shape[1] + EPS)
    out = [torch.einsum("tk,nk->tn", rows, w.double() * ws.double()[:, None]) for w, ws in s["w"]]
    if s["op"] == "swiglu":
        return out[0] * torch.sigmoid(out[0]) * out[1]
    out = out[0]
    for more in (s["bias"], s["residual"]):
        if more is not None:
            out += more.double()
    return out


def _exact_sample(s):
    rows = s["logits"].shape[0]
    own_of = {}
    for n in ("temperature", "top_k", "top_p", "min_p"):
        x = s[n] if isinstance(s[n], torch.Tensor) else torch.tensor([s[n]] * rows, dtype=torch.int32 if n == "top_k" else torch.float32)
        own_of[n] = x.tolist()
    out = torch.empty(rows, dtype=torch.float64)
    for r, (u, line) in enumerate(zip(s["uniform"].tolist(), s["logits"])):
        # only the kept ones' order matters, so the rows are cut to them one filter at a time
        value, index = torch.sort(line.double().cpu(), descending=True, stable=True)
        k, p, m, T = (own_of[n][r] for n in ("top_k", "top_p", "min_p", "temperature"))
        if k > 0:
            value = value[:k]
        score = (value - value[0]) / T
        mass = score.exp()
        if p < 1:
            sums = mass.cumsum(0)
            mass = mass[:1 + int((sums[:-1] < p * sums[-1]).sum())]
        mass = mass[mass >= m]
        sums = mass.cumsum(0)
        at = min(int(torch.searchsorted(sums, u * float(sums[-1]), right=True)), len(sums) - 1)
        out[r] = float(score[at]) - math.log(float(mass.sum()))
    return {"tokens": None, "logprob": out}
