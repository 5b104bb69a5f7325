"""What this repository's per-request logits operators are measured on.

Two operators stand between a batch's hidden states and its tokens, where
requests of one batch differ from each other:

* ``process``: penalties for repeated tokens, biases and grammar masks on the
  logits, in place (``noel_b200.sampler.logits_process``).  Row b with history
  h[0:len], of which h[0:prompt] is the prompt, and id v:
      n = occurrences of v in h[prompt:len],  seen = v occurs in h[0:len]
      x = x / rep if x > 0 else x * rep        (seen)
      x = x - freq * n - pres * (n > 0)
      x = x + sum of the row's biases on v
      x = -inf where the row's mask has a 0 bit for v
* ``lora``: low-rank adapters beside a shared projection, y already holding
  the projection (``noel_b200.sampler.lora_apply``):
      y[b] += scale[a] * B[a] (A[a] x[b]),  a = adapter[b]; a = -1: none

Both update their buffer in place, as a server does with its logits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _process(name, batch, vocab, dtype, history, ids="uniform", bias=0, masks=0, allowed=1.0, pad=0):
    return {"name": name, "op": "process", "batch": batch, "vocab": vocab, "dtype": dtype, "history": history,
            "ids": ids, "bias": bias, "masks": masks, "allowed": allowed, "pad": pad}


def _lora(name, batch, cols, rows, rank, adapters, dtype, without=0.0, ragged=False):
    return {"name": name, "op": "lora", "batch": batch, "cols": cols, "rows": rows, "rank": rank,
            "adapters": adapters, "dtype": dtype, "without": without, "ragged": ragged}


def listed():
    return [
        # one request being decoded: a short context, a few biased ids; only latency counts
        _process("process_one_row", 1, 151936, "f32", 64, bias=8),
        # a full batch under a strict grammar (a JSON key, a number): few ids are allowed
        _process("process_grammar", 1024, 152064, "f32", 64, masks=64, allowed=0.005),
        # a full batch inside grammar strings: nearly every id is allowed
        _process("process_open_bf16", 1024, 256000, "bf16", 256, masks=1024, allowed=0.98),
        # chat requests with text-like repeats and a long bias list (the usual limit of an API)
        _process("process_zipf_bias", 256, 152064, "f32", 1024, ids="zipf", bias=300),
        # long documents in the context
        _process("process_long_history", 64, 152064, "f32", 65536, ids="zipf"),
        # an odd vocabulary in rows that are wider than it, masks that allow half of the ids
        _process("process_odd_bf16", 37, 50001, "bf16", 333, ids="zipf", bias=17, masks=37, allowed=0.5, pad=7),
        # one request with an adapter on the output projection
        _lora("lora_one_token", 1, 4096, 152064, 16, 4, "bf16"),
        # a decode batch in which every request brings its own adapter
        _lora("lora_distinct", 64, 4096, 152064, 16, 64, "bf16"),
        # a decode batch over a few popular adapters of several ranks, some requests without any
        _lora("lora_shared", 256, 4096, 152064, 32, 8, "f16", without=0.25, ragged=True),
        # scoring whole prompts (every position's logits) under large adapters
        _lora("lora_scoring", 2048, 4096, 152064, 64, 4, "bf16"),
        # odd sizes throughout, full-precision adapters
        _lora("lora_odd_f32", 19, 1000, 32001, 12, 5, "f32", without=0.1),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    case = _draw_process(rng) if rng.random() < 0.5 else _draw_lora(rng)
    del case["name"]
    return case


def _draw_process(rng):
    vocab = _log_int(rng, 1000, 262144)
    batch = min(_log_int(rng, 1, 1024), max(1, 1024 * 152064 // vocab))
    masked = rng.random() < 0.6
    history = _log_int(rng, 1, min(65536, 64 * 65536 // batch))
    return _process("", batch, vocab, rng.choice(["f32", "bf16"]), history, ids=rng.choice(["uniform", "zipf"]),
                    bias=rng.choice([0, rng.randint(1, 300)]), masks=_log_int(rng, 1, batch) if masked else 0,
                    allowed=rng.choice([0.001, 0.01, 0.1, 0.5, 0.9, 0.99]) if masked else 1.0,
                    pad=rng.choice([0, 0, rng.randint(1, 64)]))


def _draw_lora(rng):
    rows = _log_int(rng, 1000, 152064)
    rank = rng.choice([_log_int(rng, 1, 64), 8, 16, 32, 64])
    batch = _log_int(rng, 1, 2048)
    adapters = min(_log_int(rng, 1, 64), max(1, 64 * 16 // rank))
    while batch * adapters > 2048 * 4 * 64 // rank:  # the plain form multiplies every token by every adapter
        batch = (batch + 1) // 2
    return _lora("", batch, _log_int(rng, 64, 8192), rows, rank, adapters, rng.choice(["f32", "f16", "bf16"]),
                 without=rng.choice([0.0, 0.3]), ragged=rng.random() < 0.3)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _zipf_ids(shape, vocab, g):
    # the law P(rank) ~ 1 / rank by inversion of its integral: id = vocab^u - 1
    u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1.0)) - 1.0).floor().clamp_(0, vocab - 1).to(torch.int32)


def _prepare_process(case, seed):
    g = _generator(seed)
    B, V, H = case["batch"], case["vocab"], case["history"]
    dev = "cuda"
    rows = torch.randn(B, V + case["pad"], generator=g, device=dev).mul_(3.0).to(DTYPES[case["dtype"]])
    history = (_zipf_ids((B, H), V, g) if case["ids"] == "zipf"
               else torch.randint(0, V, (B, H), generator=g, device=dev, dtype=torch.int32))
    lens = torch.randint((H + 1) // 2, H + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    s = {"logits": rows[:, :V], "history": history, "history_lens": lens, "prompt_lens": (lens // 2).to(torch.int32),
         "repetition": 1.0 + 0.3 * torch.rand(B, generator=g, device=dev),
         "frequency": 0.5 * torch.rand(B, generator=g, device=dev),
         "presence": 0.5 * torch.rand(B, generator=g, device=dev),
         "bias_ids": None, "bias": None, "mask": None, "mask_rows": None}
    if case["bias"]:
        s["bias_ids"] = torch.randint(0, V, (B, case["bias"]), generator=g, device=dev, dtype=torch.int32)
        s["bias"] = 2.0 * torch.randn(B, case["bias"], generator=g, device=dev)
    if case["masks"]:
        words = (V + 31) // 32
        weight = torch.ones(32, dtype=torch.int64, device=dev) << torch.arange(32, device=dev)
        bits = torch.rand(case["masks"], words, 32, generator=g, device=dev) < case["allowed"]
        s["mask"] = (bits * weight).sum(2).to(torch.int32)
        # row b under mask b mod masks; one row in sixteen is free text
        which = torch.arange(B, device=dev, dtype=torch.int32) % case["masks"]
        s["mask_rows"] = torch.where(torch.arange(B, device=dev) % 16 == 15, -1, which).to(torch.int32)
    return s


def _adapter_ids(case, g):
    B, n = case["batch"], case["adapters"]
    with_one = B - int(B * case["without"])
    ids = torch.arange(B, device="cuda", dtype=torch.int32) % n
    ids[with_one:] = -1
    return ids[torch.randperm(B, generator=g, device="cuda")].contiguous()


def _ranks(case):
    """Ranks of the adapters: all the same, or r, r/2, r/4 in turn."""
    return [max(1, case["rank"] >> (i % 3)) if case["ragged"] else case["rank"] for i in range(case["adapters"])]


def _prepare_lora(case, seed):
    g = _generator(seed)
    B, D, V, r, n = case["batch"], case["cols"], case["rows"], case["rank"], case["adapters"]
    dev, t = "cuda", DTYPES[case["dtype"]]
    return {"y": torch.randn(B, V, generator=g, device=dev).mul_(3.0),
            "x": torch.randn(B, D, generator=g, device=dev),
            "a": torch.randn(n, r, D, generator=g, device=dev).mul_(D ** -0.5).to(t),
            "b": torch.randn(n, V, r, generator=g, device=dev).mul_(0.5).to(t),
            "scale": 0.5 + torch.rand(n, generator=g, device=dev),
            "ranks": torch.tensor(_ranks(case), dtype=torch.int32, device=dev) if case["ragged"] else None,
            "adapter": _adapter_ids(case, g)}


def prepare(case, seed):
    s = _prepare_process(case, seed) if case["op"] == "process" else _prepare_lora(case, seed)
    s["op"] = case["op"]
    if own:
        # the handles that a server keeps: they hold the tensors above and nothing computed from them
        from noel_b200 import sampler as S

        if case["op"] == "process":
            s["params"] = S.LogitsParams(**{k: s[k] for k in (
                "history", "history_lens", "prompt_lens", "repetition", "frequency", "presence", "bias_ids", "bias",
                "mask", "mask_rows")})
        else:
            s["adapters"] = S.Adapters(s["a"], s["b"], scale=s["scale"], ranks=s["ranks"])
    return s


def _plain_process(s):
    logits = s["logits"]
    B, V = logits.shape
    H = s["history"].shape[1]
    at = torch.arange(H, device=logits.device)
    inside = at < s["history_lens"][:, None]
    output = inside & (at >= s["prompt_lens"][:, None])
    ids = s["history"].long()
    seen = torch.zeros(B, V, dtype=torch.int32, device=logits.device).scatter_add_(1, ids, inside.to(torch.int32))
    count = torch.zeros(B, V, dtype=torch.int32, device=logits.device).scatter_add_(1, ids, output.to(torch.int32))
    x = logits.float()
    rep = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"].long(), s["bias"])
    if s["mask"] is not None:
        v = torch.arange(V, device=logits.device)
        words = s["mask"][s["mask_rows"].clamp(min=0).long()]
        bit = (words[:, v >> 5] >> (v & 31).to(torch.int32)) & 1
        x = torch.where((bit == 1) | (s["mask_rows"] < 0)[:, None], x, float("-inf"))
    return logits.copy_(x)


def _plain_lora(s):
    n, r, _ = s["a"].shape
    mine = s["adapter"][:, None] == torch.arange(n, device=s["y"].device)  # a token times every adapter, its own kept
    low = torch.einsum("bd,nrd->bnr", s["x"], s["a"].float())
    low = low * (mine * s["scale"])[:, :, None]
    b = s["b"].float()
    if s["ranks"] is not None:
        low = low * (torch.arange(r, device=low.device) < s["ranks"][:, None])
    return s["y"].add_(torch.einsum("bnr,nvr->bv", low, b))


def run(state):
    if own:
        from noel_b200 import sampler as S

        if state["op"] == "process":
            return S.logits_process(state["logits"], state["params"])
        return S.lora_apply(state["y"], state["x"], state["adapters"], state["adapter"])
    return _plain_process(state) if state["op"] == "process" else _plain_lora(state)


def _distinct(case):
    """Expected number of different ids in a row's history of 3/4 of its full length."""
    V, n = case["vocab"], 0.75 * case["history"]
    if case["ids"] == "uniform":
        return V * -math.expm1(n * math.log1p(-1.0 / V)) if V > 1 else 1.0
    v = torch.arange(V, dtype=torch.float64)
    p = torch.log1p(1.0 / (v + 1.0)) / math.log(V + 1.0)
    return float((-torch.expm1(n * torch.log1p(-p))).sum())


def work(case):
    B = case["batch"]
    if case["op"] == "process":
        V, es = case["vocab"], 4 if case["dtype"] == "f32" else 2
        free = B // 16 if case["masks"] else B
        masked = (B - free) * (1.0 - case["allowed"]) * V
        share = (free + (B - free) * case["allowed"]) / B  # of the ids, those that no mask takes away
        touched = B * share * (_distinct(case) + case["bias"])
        read = B * (0.75 * case["history"] * 4 + case["bias"] * 8 + 24) + case["masks"] * ((V + 31) // 32) * 4
        return {"bytes": read + 2 * touched * es + masked * es, "flops": 6 * touched}
    D, V = case["cols"], case["rows"]
    es = 4 if case["dtype"] == "f32" else 2
    tokens = B - int(B * case["without"])
    ranks = _ranks(case)
    used = ranks[:min(tokens, case["adapters"])]
    mean = sum(ranks[i % len(ranks)] for i in range(tokens)) / max(1, tokens)
    return {"bytes": tokens * (D * 4 + 2 * V * 4) + B * 4 + sum(used) * (D + V) * es,
            "flops": 2 * tokens * mean * (D + V)}


def _exact_process(case, seed):
    s = _prepare_process(case, seed)
    x = s["logits"].double()
    B, V = x.shape
    # row by row, from the list of the row's different ids and how often each occurs
    for b in range(B):
        h = s["history"][b, :int(s["history_lens"][b])].long()
        seen = torch.unique(h)
        rep = s["repetition"][b].double()
        old = x[b, seen]
        x[b, seen] = torch.where(old > 0, old / rep, old * rep)
        out, times = torch.unique(h[int(s["prompt_lens"][b]):], return_counts=True)
        x[b, out] -= s["frequency"][b].double() * times.double() + s["presence"][b].double()
    if s["bias"] is not None:
        for k in range(case["bias"]):
            at = s["bias_ids"][:, k:k + 1].long()
            x.scatter_(1, at, x.gather(1, at) + s["bias"][:, k:k + 1].double())
    if s["mask"] is not None:
        for bit in range(32):
            part = x[:, bit::32]
            gone = (s["mask"][:, :part.shape[1]] >> bit & 1) == 0
            rows = s["mask_rows"].long()
            part.masked_fill_(gone[rows.clamp(min=0)] & (rows >= 0)[:, None], float("-inf"))
    return x


def _exact_lora(case, seed):
    s = _prepare_lora(case, seed)
    y = s["y"].double()
    for i, r in enumerate(_ranks(case)):
        tokens = (s["adapter"] == i).nonzero()[:, 0]
        if tokens.numel():
            low = s["x"][tokens].double() @ s["a"][i, :r].double().T
            y[tokens] += s["scale"][i].double() * (low @ s["b"][i, :, :r].double().T)
    return y


def exact(case, seed):
    return _exact_process(case, seed) if case["op"] == "process" else _exact_lora(case, seed)
