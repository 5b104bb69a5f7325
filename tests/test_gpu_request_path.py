"""The per-request operators together, as a server runs them: the LM head,
each token's adapter, penalties / biases / masks, and the sampler, in one call;
and processed shards through the vocab-sharded sampler."""
import numpy as np
import pytest

from tests.request_ops import lora_plain, process_plain, within
from tests.test_gpu_logits import build as process_inputs
from tests.test_gpu_logits import params

pytestmark = pytest.mark.gpu

CFG = dict(temperature=0.8, top_p=0.95, top_k=40, repetition_penalty=1.0)


def inputs(cuda, B, D=512, V=9000, r=16, n=3, seed=0):
    import torch

    g = torch.Generator(device=cuda).manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    _, p = process_inputs(B, V, "f32", seed=seed, H=200, bias=12, masks=min(B, 4), density=0.4)
    if "mask_rows" in p:
        p["mask_rows"][p["mask_rows"] == 1] = -1  # the mask that allows nothing
    return {"weight": (f(V, D) * 0.05).to(torch.bfloat16), "hidden": f(B, D),
            "a": (f(n, r, D) * D ** -0.5).to(torch.bfloat16), "b": (f(n, V, r) * 0.5).to(torch.bfloat16),
            "ids": torch.randint(-1, n, (B,), generator=g, device=cuda, dtype=torch.int32),
            "rng": torch.randint(1, 2**62, (B, 2), generator=g, device=cuda, dtype=torch.int64), "process": p}


def double(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("B", [1, 5, 8, 21])
def test_head_adapters_processing_sampler_gpu(cuda, B):
    import torch

    from noel_b200 import sampler as S

    s = inputs(cuda, B, seed=B)
    cfg = S.make_config(**CFG)
    ad, prm = S.Adapters(s["a"], s["b"]), params(S, cuda, s["process"])
    rng = s["rng"].clone()
    ids, logits, probs = S.lmhead_sample(s["weight"], s["hidden"], rng, cfg, probs=True, adapters=ad,
                                         adapter_ids=s["ids"], process=prm)
    # the plain projection, whose bits the head's own tests pin
    _, base, _ = S.lmhead_sample(s["weight"], s["hidden"], s["rng"].clone(), cfg)
    mid, mid_bound = lora_plain(double(base), double(s["hidden"]), double(s["a"]), double(s["b"]), s["ids"].cpu().numpy())
    want, bound, _ = process_plain(mid, **s["process"])
    # processing multiplies an error by at most the repetition penalty (1.4 at most), then adds its own; a value within its
    # error of 0 may be divided on one side and multiplied on the other, which moves it by no more than twice that error
    reach = 2.0 * mid_bound
    within(logits.double().cpu().numpy(), want, np.where(np.isfinite(want), bound + reach, 0.0))
    # the tokens are the sampler's on those logits
    rng2 = s["rng"].clone()
    out = S.sample_batch(logits.clone(), rng2, cfg)
    assert torch.equal(ids, out["ids"]) and torch.equal(probs, out["probs"]) and torch.equal(rng, rng2)
    # and they are allowed ones
    p = s["process"]
    for b, t in enumerate(ids.tolist()):
        m = p["mask_rows"][b]
        if 0 <= m < len(p["mask"]):
            assert p["mask"][m, t >> 5] >> (t & 31) & 1


def test_the_steps_one_by_one_give_the_same_bits_gpu(cuda):
    import torch

    from noel_b200 import sampler as S

    s = inputs(cuda, 13, seed=40)
    cfg = S.make_config(**CFG)
    ad, prm = S.Adapters(s["a"], s["b"]), params(S, cuda, s["process"])
    ids, logits, _ = S.lmhead_sample(s["weight"], s["hidden"], s["rng"].clone(), cfg, adapters=ad, adapter_ids=s["ids"],
                                     process=prm)
    _, y, _ = S.lmhead_sample(s["weight"], s["hidden"], s["rng"].clone(), cfg)
    S.logits_process(S.lora_apply(y, s["hidden"], ad, s["ids"]), prm)
    assert torch.equal(y, logits)
    assert torch.equal(S.sample_batch(y, s["rng"].clone(), cfg)["ids"], ids)


def test_two_graphs_of_the_path_gpu(cuda):
    """the whole path captured twice, replayed in turn and at once on two streams"""
    import torch

    from noel_b200 import sampler as S

    cfg = S.make_config(**CFG)
    made = []
    for seed in (1, 2):
        s = inputs(cuda, 9, seed=seed)
        ad, prm = S.Adapters(s["a"], s["b"]), params(S, cuda, s["process"])
        stream = torch.cuda.Stream()
        args = dict(adapters=ad, adapter_ids=s["ids"], process=prm)
        rng0 = s["rng"].clone()
        with torch.cuda.stream(stream):  # the sampler's scratch is made by a call before the capture
            want = S.lmhead_sample(s["weight"], s["hidden"], s["rng"], cfg, **args)[:2]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            got = S.lmhead_sample(s["weight"], s["hidden"], s["rng"], cfg, **args)[:2]
        made.append((g, stream, s, rng0, want, got, args))
    for _ in range(3):
        for g, stream, s, rng0, want, got, _ in made:
            s["rng"].copy_(rng0)
        torch.cuda.synchronize()
        for g, stream, *_ in made:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for g, stream, s, rng0, want, got, _ in made:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_processed_shards_through_the_sharded_sampler_gpu(cuda):
    import torch

    from noel_b200 import sampler as S
    from noel_b200 import sharded

    B, V = 8, 6000
    t, p = process_inputs(B, V, "f32", seed=77, H=100, bias=10, masks=B, density=0.2)
    p["mask_rows"][p["mask_rows"] == 1] = -1
    cfg = S.make_config(**CFG)
    rng = torch.arange(1, 2 * B + 1, dtype=torch.int64, device=cuda).view(B, 2)
    whole = S.logits_process(t.to(cuda), params(S, cuda, p))
    want = S.sample_batch(whole, rng.clone(), cfg)["ids"]
    parts, bounds = t.to(cuda), sharded.shard_bounds(V, 3)
    for lo, width in bounds:
        S.logits_process(parts[:, lo:lo + width], params(S, cuda, p, v_begin=lo))
    got, _, _ = sharded.sample_vocab_sharded_local(cfg, parts, bounds, rng.clone())
    assert torch.equal(got, want)


def test_empty_batches_gpu(cuda):
    import torch

    from noel_b200 import sampler as S

    z = torch.zeros(0, 500, device=cuda)
    h = torch.zeros(0, 7, dtype=torch.int32, device=cuda)
    assert S.logits_process(z, S.LogitsParams(history=h)).shape == (0, 500)
    ad = S.Adapters(torch.zeros(2, 4, 16, device=cuda), torch.zeros(2, 500, 4, device=cuda))
    ids = torch.zeros(0, dtype=torch.int32, device=cuda)
    assert S.lora_apply(z, torch.zeros(0, 16, device=cuda), ad, ids).shape == (0, 500)
    x = torch.randn(3, 500, device=cuda)
    none = S.LogitsParams(history=torch.zeros(3, 0, dtype=torch.int32, device=cuda),
                          bias_ids=torch.zeros(3, 0, dtype=torch.int32, device=cuda), bias=torch.zeros(3, 0, device=cuda))
    assert torch.equal(S.logits_process(x.clone(), none), x)


def test_a_row_that_allows_nothing_is_sampled_gpu(cuda, oracle):
    """-infinity throughout goes through the sampler as it does through the reference's"""
    import torch

    from noel_b200 import sampler as S
    from oracle.oracle import make_config as orc_config

    x = torch.randn(4, 3000, device=cuda)
    S.logits_process(x, S.LogitsParams(mask=torch.zeros(1, 94, dtype=torch.int32, device=cuda),
                                       mask_rows=torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device=cuda)))
    assert torch.isneginf(x[1:3]).all() and torch.isfinite(x[[0, 3]]).all()
    rng = np.arange(1, 9, dtype=np.uint64).reshape(4, 2)
    rng_t = torch.from_numpy(rng.view(np.int64).copy()).to(cuda)
    got = S.sample_batch(x, rng_t, S.make_config(**CFG))
    want = oracle.sample_batch(orc_config(**CFG, repetition_window=0), x.cpu().numpy(), rng=rng)
    np.testing.assert_array_equal(got["ids"].cpu().numpy(), want.ids)


def test_requests_change_between_replays_gpu(cuda):
    """one captured step, replayed while the histories, biases, masks and adapters in its buffers change"""
    import torch

    from noel_b200 import sampler as S

    s = inputs(cuda, 9, seed=5)
    ad, prm = S.Adapters(s["a"], s["b"]), params(S, cuda, s["process"])
    x0, y = torch.randn(9, 9000, device=cuda), torch.empty(9, 9000, device=cuda)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y.copy_(x0)
        S.logits_process(S.lora_apply(y, s["hidden"], ad, s["ids"]), prm)
    for k in range(3):
        for t in prm.tensors:  # the buffers that the parameters were made over
            if t.dtype == torch.int32 and t.dim() == 2:
                t.copy_(t.roll(k, 0))
        s["ids"].copy_(s["ids"].roll(1))
        g.replay()
        want = S.logits_process(S.lora_apply(x0.clone(), s["hidden"], ad, s["ids"]), prm)
        assert torch.equal(y, want)


def test_path_refusals_gpu(cuda):
    import torch

    from noel_b200 import sampler as S

    s = inputs(cuda, 4, seed=3)
    cfg = S.make_config(**CFG)
    ad = S.Adapters(s["a"], s["b"])
    small = S.Adapters(s["a"], s["b"][:, :8000])
    h = torch.zeros(5, 3, dtype=torch.int32, device=cuda)
    for kw in (dict(adapters=ad), dict(adapter_ids=s["ids"]), dict(adapters=small, adapter_ids=s["ids"]),
               dict(adapters=ad, adapter_ids=s["ids"][:3]), dict(process=S.LogitsParams(history=h))):
        with pytest.raises(S.NoelSamplerError):
            S.lmhead_sample(s["weight"], s["hidden"], s["rng"], cfg, **kw)
