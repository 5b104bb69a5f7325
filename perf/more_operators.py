"""What this repository's operators between 8-bit output weights and sampled tokens are measured on.

Two operators, used one after the other by a server that keeps its output
projection in 8 bits and samples every request with its own settings:

* ``linear``: y = x W^T with both in 8-bit integers (``noel_b200.sampler.int8_linear``).
  Weights come with a scale for each output channel; tokens are cast in the call, with a scale for each token:
      s[t] = max(max_d |x[t, d]| / 127, 2^-126) in 32 bits,  q[t, d] = x[t, d] / s[t] to the nearest integer, ties to even
      y[t, v] = s[t] * w_scale[v] * sum_d q[t, d] * w[v, d]
* ``sample``: one id from each row of logits, under the row's own temperature, top-k, top-p and min-p and its own
  random number u in [0, 1) (``noel_b200.sampler.sample_requests``).  With m the row's largest logit and T its
  temperature (T <= 0: the id of m, the lowest of several):
      left are the ids with x >= m - 30 T and x >= m + T ln(min_p)            (min_p <= 0: the former only)
      of those the first k by (x descending, id ascending)                    (k <= 0: all)
      of those, in that order, the fewest whose weights exp((x - m) / T) sum to at least top_p times all of theirs
      the lowest id of those at which their weights' running sum, in the order of ids, exceeds u times their sum
  Outputs are the ids and their probabilities among what is left.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _linear(name, tokens, cols, rows, x, y, idle=0.0):
    return {"name": name, "op": "linear", "tokens": tokens, "cols": cols, "rows": rows, "x": x, "y": y, "idle": idle}


def _sample(name, batch, vocab, dtype, settings, masked=0.0, pad=0):
    return {"name": name, "op": "sample", "batch": batch, "vocab": vocab, "dtype": dtype, "settings": settings,
            "masked": masked, "pad": pad}


def listed():
    return [
        # one request being decoded: its logits
        _linear("linear_one_token", 1, 4096, 152064, "bf16", "f32"),
        # a decode batch
        _linear("linear_decode", 64, 4096, 152064, "bf16", "f32"),
        # a large decode batch, hidden states in half precision, logits to be sampled in bf16
        _linear("linear_batch_f16", 256, 4096, 152064, "f16", "bf16"),
        # scoring whole prompts: every position's logits
        _linear("linear_scoring", 2048, 4096, 152064, "bf16", "f32"),
        # a square projection inside a layer, over a prompt
        _linear("linear_prompt_layer", 4096, 4096, 4096, "bf16", "bf16"),
        # odd sizes throughout, full-precision hidden states, some of the batch's tokens are padding (zeros)
        _linear("linear_odd_f32", 23, 1000, 32001, "f32", "f32", idle=0.2),
        # one request being decoded with the usual chat settings
        _sample("sample_one_row", 1, 151936, "f32", "chat"),
        # a server's batch: every request has its own settings, some are greedy
        _sample("sample_mixed", 256, 152064, "f32", "mixed"),
        # a full batch of such requests
        _sample("sample_mixed_full", 1024, 152064, "f32", "mixed"),
        # a full batch of nucleus requests (no top-k) over bf16 logits
        _sample("sample_nucleus_bf16", 1024, 256000, "bf16", "nucleus"),
        # open-ended writing: high temperatures under min-p alone
        _sample("sample_min_p", 64, 131072, "f32", "min_p"),
        # an odd vocabulary in rows wider than it, half of it masked; plain draws from all that is allowed
        _sample("sample_open_odd_bf16", 37, 50001, "bf16", "open", masked=0.5, pad=7),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    case = _draw_linear(rng) if rng.random() < 0.5 else _draw_sample(rng)
    del case["name"]
    return case


def _draw_linear(rng):
    tokens, cols, rows = _log_int(rng, 1, 4096), _log_int(rng, 64, 8192), _log_int(rng, 256, 152064)
    while tokens * cols * rows > 2048 * 4096 * 152064 or tokens * rows > 2048 * 152064 or cols * rows > 4096 * 152064:
        tokens, cols, rows = (tokens + 1) // 2, (cols + 1) // 2 + 31, (rows + 1) // 2 + 127
    return _linear("", tokens, cols, rows, rng.choice(["f32", "f16", "bf16"]), rng.choice(["f32", "bf16"]),
                   idle=rng.choice([0.0, 0.0, 0.3]))


def _draw_sample(rng):
    vocab = _log_int(rng, 1000, 262144)
    batch = min(_log_int(rng, 1, 1024), max(1, 1024 * 152064 // vocab))
    return _sample("", batch, vocab, rng.choice(["f32", "bf16"]),
                   rng.choice(["chat", "mixed", "mixed", "nucleus", "min_p", "open"]),
                   masked=rng.choice([0.0, 0.0, 0.5, 0.99]), pad=rng.choice([0, 0, rng.randint(1, 64)]))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_linear(case, seed):
    g = _generator(seed)
    T, D, V, dev = case["tokens"], case["cols"], case["rows"], "cuda"
    x = torch.randn(T, D, generator=g, device=dev)
    # a few channels of hidden states are much larger than the others
    x = x * (1.0 + 15.0 * (torch.rand(D, generator=g, device=dev) < 0.01))
    if case["idle"]:
        x[T - int(T * case["idle"]):] = 0.0
    # weights as their cast leaves them: every channel reaches 127; rows start on 16 bytes
    pitch = (D + 15) // 16 * 16
    w = torch.zeros(V, pitch, dtype=torch.int8, device=dev)
    w_scale = torch.empty(V, device=dev)
    for at in range(0, V, 16384):
        part = torch.randn(min(16384, V - at), D, generator=g, device=dev)
        top = part.abs().amax(1)
        w[at:at + 16384, :D] = torch.round(part * (127.0 / top)[:, None]).to(torch.int8)
        w_scale[at:at + 16384] = top * (D ** -0.5 / 127.0)
    return {"x": x.to(DTYPES[case["x"]]), "w": w[:, :D], "w_scale": w_scale, "y": DTYPES[case["y"]]}


def _settings(case, g):
    """temperature, top-k, top-p and min-p of every row."""
    B, dev = case["batch"], "cuda"

    def rand():
        return torch.rand(B, generator=g, device=dev)

    def pick(*values):
        at = torch.randint(0, len(values), (B,), generator=g, device=dev)
        return torch.tensor(values, device=dev)[at]

    s = {"temperature": torch.ones(B, device=dev), "top_k": None, "top_p": None, "min_p": None}
    if case["settings"] == "chat":
        s.update(temperature=0.5 + 0.5 * rand(), top_k=pick(20, 40, 50).to(torch.int32), top_p=pick(0.8, 0.9, 0.95))
    elif case["settings"] == "mixed":
        s.update(temperature=pick(0.0, 0.6, 0.7, 0.8, 1.0, 1.2), top_k=pick(0, 0, 20, 40, 50, 1000).to(torch.int32),
                 top_p=pick(0.8, 0.9, 0.95, 1.0), min_p=pick(0.0, 0.0, 0.05, 0.1))
    elif case["settings"] == "nucleus":
        s.update(temperature=0.6 + 0.4 * rand(), top_p=pick(0.8, 0.9, 0.95))
    elif case["settings"] == "min_p":
        s.update(temperature=1.0 + 0.5 * rand(), min_p=pick(0.02, 0.05, 0.1))
    return s


def _prepare_sample(case, seed):
    g = _generator(seed)
    B, V, dev = case["batch"], case["vocab"], "cuda"
    # the weights of a model's next tokens fall with their rank r about as r^-a, and ranks lie anywhere among the ids:
    # with u uniform, u V is such a rank and the logit is -a ln(u V); a is larger where the model is surer
    a = 1.3 + 1.7 * torch.rand(B, 1, generator=g, device=dev)
    rows = torch.rand(B, V + case["pad"], generator=g, device=dev)
    rows = rows.clamp_(min=2.0 ** -25).mul_(V).log_().mul_(-a).add_(8.0)
    if case["masked"]:
        gone = torch.rand(B, V, generator=g, device=dev) < case["masked"]
        gone[:, 0] = False
        rows[:, :V].masked_fill_(gone, float("-inf"))
    s = {"logits": rows.to(DTYPES[case["dtype"]])[:, :V]}
    s["u"] = torch.rand(B, generator=g, device=dev)
    s.update(_settings(case, g))
    return s


def prepare(case, seed):
    s = _prepare_linear(case, seed) if case["op"] == "linear" else _prepare_sample(case, seed)
    s["op"] = case["op"]
    if own:
        # the handles that a server keeps: they hold the tensors above and nothing computed from them
        from noel_b200 import sampler as S

        if case["op"] == "linear":
            s["weight"] = S.Int8Rows(s["w"], s["w_scale"])
        else:
            s["params"] = S.SampleParams(**{k: s[k] for k in ("temperature", "top_k", "top_p", "min_p")})
    return s


def _plain_linear(s):
    x = s["x"].float()
    scale = x.abs().amax(1)
    scale = (scale / torch.full_like(scale, 127.0)).clamp_(min=2.0 ** -126)  # divided, not times 1 / 127
    # in 64 bits no quotient of two fp32 numbers is rounded onto a half
    q = torch.round(x.double() / scale.double()[:, None]).float()
    return (q @ s["w"].float().T * scale[:, None] * s["w_scale"]).to(s["y"])


def _plain_sample(s):
    parts = [_plain_sample_rows(s, at, at + 64) for at in range(0, s["logits"].shape[0], 64)]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def _plain_sample_rows(s, begin, end):
    # in 64 bits: the draw goes by which side of a border a sum is on
    def of(name):
        return s[name][begin:end, None].double() if s[name] is not None else None

    x = s["logits"][begin:end].double()
    B, V = x.shape
    top = x.amax(1, keepdim=True)
    greedy = of("temperature") <= 0
    t = torch.where(greedy, torch.ones_like(top), of("temperature"))
    x, ids = torch.sort(x, dim=1, descending=True, stable=True)
    left = x >= top - 30.0 * t
    if s["min_p"] is not None:
        p = of("min_p")
        left &= (x >= top + t * torch.log(p)) | (p <= 0)
    at = torch.arange(V, device=x.device)
    if s["top_k"] is not None:
        k = s["top_k"][begin:end, None]
        left &= (at < k) | (k <= 0)
    left &= (at < 1) | ~greedy
    w = torch.where(left, torch.exp((x - top) / t), torch.zeros_like(x))
    if s["top_p"] is not None:
        p = of("top_p")
        before = torch.cumsum(w, 1) - w
        w = torch.where((before < p * w.sum(1, keepdim=True)) | (p >= 1) | (at < 1), w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, ids, w)  # back in the order of ids
    run = torch.cumsum(w, 1)
    total = run[:, -1:]
    over = (run > of("u") * total) & (w > 0)
    drawn = torch.where(over, at, V - 1).amin(1, keepdim=True)
    return drawn[:, 0].to(torch.int32), (w.gather(1, drawn) / total)[:, 0].float()


def run(state):
    if own:
        from noel_b200 import sampler as S

        if state["op"] == "linear":
            return S.int8_linear(state["x"], state["weight"], dtype=state["y"])
        return S.sample_requests(state["logits"], state["u"], state["params"])
    return _plain_linear(state) if state["op"] == "linear" else _plain_sample(state)


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "linear":
        T, D, V = case["tokens"], case["cols"], case["rows"]
        return {"bytes": T * D * size[case["x"]] + V * D + 4 * V + T * V * size[case["y"]], "flops": 2 * T * D * V}
    B, V = case["batch"], case["vocab"]
    # a row's logits once, its number and settings, its id and probability; a comparison an id
    given = {"chat": 3, "mixed": 4, "nucleus": 2, "min_p": 2, "open": 1}[case["settings"]]
    return {"bytes": B * (V * size[case["dtype"]] + 4 * (1 + given) + 8), "flops": B * V}


def _exact_linear(case, seed):
    if case["tokens"] * case["cols"] * case["rows"] > 2 ** 41:
        return None
    s = _prepare_linear(case, seed)
    x = s["x"].double()
    scale = (x.abs().amax(1) / 127.0).float().double().clamp(min=2.0 ** -126)
    below = torch.floor(x / scale[:, None])
    twice = 2.0 * (x - below * scale[:, None])  # against one step, exactly: the numbers have 32 bits at most
    odd = torch.remainder(below, 2.0) == 1.0
    up = (twice > scale[:, None]) | ((twice == scale[:, None]) & odd)
    q = below + up
    y = torch.empty(case["tokens"], case["rows"], dtype=torch.float64, device="cuda")
    for v in range(0, case["rows"], 8192):
        y[:, v:v + 8192] = q @ s["w"][v:v + 8192].double().T
    return y * (scale[:, None] * s["w_scale"].double())


def _exact_sample(case, seed):
    s = _prepare_sample(case, seed)
    B = case["batch"]

    def values(name, off):
        return s[name].double().tolist() if s[name] is not None else [off] * B

    drawn, probs = [], []
    settings = zip(values("temperature", 1.0), values("top_k", 0), values("top_p", 1.0), values("min_p", 0.0),
                   values("u", 0.0))
    # row by row, from the list of the ids that are left
    for b, (t, k, p, least, u) in enumerate(settings):
        x = s["logits"][b].double()
        m = x.max()
        if t <= 0:
            drawn.append((x == m).nonzero()[0, 0])
            probs.append(torch.ones((), dtype=torch.float64, device="cuda"))
            continue
        floor = m + t * max(-30.0, math.log(least) if least > 0 else -math.inf)
        ids = (x >= floor).nonzero()[:, 0]
        order = torch.argsort(x[ids], descending=True, stable=True)
        if k > 0:
            order = order[:int(k)]
        w = torch.exp((x[ids[order]] - m) / t)
        if p < 1:
            n = torch.searchsorted(torch.cumsum(w, 0), p * w.sum()) + 1
            keep = torch.arange(w.numel(), device="cuda") < n
            order, w = order[keep], w[keep]
        place = torch.argsort(order)
        run = torch.cumsum(w[place], 0)
        at = (run <= u * run[-1]).sum().clamp(max=run.numel() - 1)
        drawn.append(ids[order[place[at]]])
        probs.append(w[place[at]] / run[-1])
    return torch.stack(drawn).to(torch.int32), torch.stack(probs)


def exact(case, seed):
    return _exact_linear(case, seed) if case["op"] == "linear" else _exact_sample(case, seed)
