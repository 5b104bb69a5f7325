"""Sampling with every row's own settings on the GPU (include/noel_requests.h)
against its definition in 64 bits: ids and counts equal, probabilities to
their last rounding."""
import numpy as np
import pytest

from tests.request_sampling import sample_plain

pytestmark = pytest.mark.gpu

# A probability is exp(d) / total in 64 bits, rounded once to fp32 (2^-24).  The kernel's total is a sum of weights of
# which each is off by 2^-44 of the largest weight at most, so the total of n by n 2^-44: below 2^-24 for n < 2^20.
PROB_RTOL = 2.0**-24 + 2.0**-24


def rows_of(rng, batch, vocab, kind):
    if kind == "normal":
        return (rng.standard_normal((batch, vocab)) * 3).astype(np.float32)
    if kind == "flat":
        return (rng.standard_normal((batch, vocab)) * 0.25).astype(np.float32)
    if kind == "ties":
        return rng.integers(-6, 7, (batch, vocab)).astype(np.float32)
    if kind == "zipf":
        a = rng.uniform(1.2, 3.0, (batch, 1))
        return (8.0 - a * np.log(np.maximum(rng.uniform(size=(batch, vocab)), 2.0**-25) * vocab)).astype(np.float32)
    if kind == "masked":
        x = (rng.standard_normal((batch, vocab)) * 2).astype(np.float32)
        x[rng.uniform(size=x.shape) < 0.9] = -np.inf
        x[rng.uniform(size=x.shape) < 0.01] = np.nan
        return x
    raise KeyError(kind)


def settings_of(rng, batch, vocab):
    """Every combination of settings that are on and off, and of their extremes, over the rows."""
    t = rng.choice(np.array([0.0, 0.3, 0.7, 1.0, 1.0, 1.5, 5.0], np.float32), batch)
    k = rng.choice(np.array([0, 0, 1, 2, 40, 50, 1000, vocab - 1, vocab, 2**31 - 1]), batch).astype(np.int32)
    p = rng.choice(np.array([1.0, 1.0, 0.0, 1e-6, 0.5, 0.9, 0.95, 0.999999, 2.0], np.float32), batch)
    q = rng.choice(np.array([0.0, 0.0, 1e-9, 0.001, 0.05, 0.5, 1.0, 3.0], np.float32), batch)
    return t, k, p, q


def check(x, u, names, values, dtype="float32", pad=0, dev=None):
    import torch

    from noel_b200 import sampler as S

    full = np.full((x.shape[0], x.shape[1] + pad), 1e30, np.float32)
    full[:, :x.shape[1]] = x
    logits = torch.from_numpy(full).to(dev, getattr(torch, dtype))
    before = logits.clone()
    params = S.SampleParams(**{n: torch.from_numpy(v).to(dev) for n, v in zip(names, values)})
    ids, probs, counts = S.sample_requests(logits, torch.from_numpy(u).to(dev), params, vocab=x.shape[1], counts=True)
    want = sample_plain(logits[:, :x.shape[1]].float().cpu().numpy(), u, **dict(zip(names, values)))
    np.testing.assert_array_equal(counts.cpu().numpy(), want[2])
    np.testing.assert_array_equal(ids.cpu().numpy(), want[0])
    np.testing.assert_allclose(probs.cpu().numpy(), want[1], rtol=PROB_RTOL, atol=0)
    assert torch.equal(logits.view(torch.int32 if dtype == "float32" else torch.int16),
                       before.view(torch.int32 if dtype == "float32" else torch.int16))


NAMES = ("temperature", "top_k", "top_p", "min_p")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kind", ["normal", "flat", "ties", "zipf", "masked"])
@pytest.mark.parametrize("batch,vocab,pad", [(1, 1, 0), (5, 2, 1), (40, 33, 0), (70, 1000, 3), (64, 4097, 0), (33, 32000, 0),
                                             (20, 50001, 7), (400, 5000, 0)])
def test_mixed_settings(cuda, dtype, kind, batch, vocab, pad):
    rng = np.random.default_rng(batch * 131 + vocab)
    x = rows_of(rng, batch, vocab, kind)
    u = rng.uniform(size=batch).astype(np.float32)
    check(x, u, NAMES, settings_of(rng, batch, vocab), dtype, pad, cuda)


@pytest.mark.parametrize("batch,vocab", [(1, 152064), (17, 152064), (330, 100003)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kind", ["zipf", "flat"])
def test_large_vocabularies(cuda, batch, vocab, dtype, kind):
    rng = np.random.default_rng(batch)
    x = rows_of(rng, batch, vocab, kind)
    check(x, rng.uniform(size=batch).astype(np.float32), NAMES, settings_of(rng, batch, vocab), dtype, 0, cuda)


def test_rows_beyond_the_shared_memory(cuda):
    rng = np.random.default_rng(3)
    for vocab in (700001, 1048576):
        x = rows_of(rng, 4, vocab, "zipf")
        check(x, rng.uniform(size=4).astype(np.float32), NAMES, settings_of(rng, 4, vocab), "float32", 0, cuda)


@pytest.mark.parametrize("name", NAMES)
def test_one_setting_alone(cuda, name):
    rng = np.random.default_rng(8)
    batch, vocab = 60, 3001
    values = dict(zip(NAMES, settings_of(rng, batch, vocab)))
    check(rows_of(rng, batch, vocab, "normal"), rng.uniform(size=batch).astype(np.float32), (name,), (values[name],),
          dev=cuda)


def test_no_settings(cuda):
    rng = np.random.default_rng(9)
    check(rows_of(rng, 50, 9999, "normal"), rng.uniform(size=50).astype(np.float32), (), (), dev=cuda)


def test_uniforms_at_their_ends(cuda):
    rng = np.random.default_rng(10)
    u = np.array([0.0, -1.0, np.nan, 1.0 - 2.0**-24, 1.0, 7.0, np.inf, 1e-45, 2.0**-30], np.float32)
    x = np.repeat(rows_of(rng, 1, 2000, "normal"), len(u), 0)
    for t in (0.2, 1.0, 100.0):
        check(x, u, ("temperature",), (np.full(len(u), t, np.float32),), dev=cuda)


def test_odd_rows_and_settings(cuda):
    nan, inf = np.nan, np.inf
    x = np.array([[-inf, -inf, -inf, -inf], [nan, nan, nan, nan], [-inf, nan, 2.0, -inf], [1.0, inf, 0.0, inf],
                  [inf, inf, nan, 3.0], [-3.4e38, 3.4e38, 0.0, 1.0], [0.0, -0.0, 0.0, -0.0], [1e-45, 0.0, -1e-45, 2e-45],
                  [-inf, -3.4e38, -3.4e38, -inf], [5.0, 5.0, 5.0, 5.0]], np.float32)
    settings = [(t, k, p, q) for t in (-1.0, 0.0, nan, 1e-45, 1e-6, 1.0, 3e38, inf) for k in (-5, 0, 1, 2, 3, 4)
                for p in (-1.0, 0.0, 0.4, 1.0, nan) for q in (-1.0, 0.0, 1e-30, 0.3, 1.0, 2.0, nan)]
    t, k, p, q = (np.repeat(np.array(c, np.float32), len(x)) for c in zip(*settings))
    big = np.tile(x, (len(settings), 1))
    u = np.random.default_rng(11).uniform(size=len(big)).astype(np.float32)
    check(big, u, NAMES, (t, k.astype(np.int32), p, q), dev=cuda)


def test_ties_at_the_cut_go_by_id(cuda):
    vocab = 20000
    x = np.zeros((6, vocab), np.float32)
    x[:, 5000:5003] = 1.0
    x[3:, ::2] = -1.0
    k = np.array([1, 2, 3, 4, 9000, 19999], np.int32)
    rng = np.random.default_rng(12)
    for _ in range(8):
        check(x, rng.uniform(size=6).astype(np.float32), ("top_k",), (k,), dev=cuda)
    p = np.array([1e-9, 0.1, 0.25, 0.5, 0.75, 0.99], np.float32)
    for _ in range(8):
        check(x, rng.uniform(size=6).astype(np.float32), ("top_p",), (p,), dev=cuda)


def test_results_do_not_depend_on_the_batch(cuda):
    import torch

    from noel_b200 import sampler as S

    rng = np.random.default_rng(13)
    B, V = 500, 12345
    logits = torch.from_numpy(rows_of(rng, B, V, "zipf")).to(cuda)
    u = torch.from_numpy(rng.uniform(size=B).astype(np.float32)).to(cuda)
    values = [torch.from_numpy(v).to(cuda) for v in settings_of(rng, B, V)]
    ids, probs, counts = S.sample_requests(logits, u, S.SampleParams(*values), counts=True)
    for at, n in ((0, 1), (7, 20), (100, 333)):
        part = S.sample_requests(logits[at:at + n], u[at:at + n], S.SampleParams(*(v[at:at + n] for v in values)), counts=True)
        for got, whole in zip(part, (ids, probs, counts)):
            assert torch.equal(got, whole[at:at + n])


def test_graphs_share_nothing(cuda):
    """Two captured calls replayed in turn, on new logits each time, and a stream other than the current one."""
    import torch

    from noel_b200 import sampler as S

    rng = np.random.default_rng(14)
    calls = []
    for B, V in ((3, 40000), (400, 3000)):
        logits, u = torch.empty(B, V, device=cuda), torch.empty(B, device=cuda)
        params = S.SampleParams(*(torch.from_numpy(v).to(cuda) for v in settings_of(rng, B, V)))
        S.sample_requests(logits.zero_(), u.zero_(), params)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = S.sample_requests(logits, u, params, counts=True)
        calls.append((logits, u, params, g, out))
    side = torch.cuda.Stream()
    for turn in range(4):
        for logits, u, *_ in calls:
            logits.normal_().mul_(3)
            u.uniform_()
        for *_, g, _ in calls:
            g.replay()
        torch.cuda.synchronize()
        for logits, u, params, _, out in calls:
            again = S.sample_requests(logits, u, params, counts=True, stream=side)
            side.synchronize()
            for x, y in zip(out, again):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch", [30, 700])
def test_odd_values_in_large_rows(cuda, dtype, batch):
    """Infinities, NaN, masks of the type's lowest value and rows with nothing, under all kinds of settings; with 700
    rows a CTA has a row of its own."""
    rng = np.random.default_rng(21)
    vocab = 20011
    x = rows_of(rng, batch, vocab, "zipf")
    low = np.float32(-3.3895314e38) if dtype == "bfloat16" else np.float32(-3.4028235e38)
    kind = np.arange(batch) % 10
    x[kind == 1, 15000:15003] = np.inf
    x[kind == 2, ::7] = np.nan
    x[kind == 3, :] = np.where(rng.uniform(size=vocab) < 0.999, low, x[kind == 3, :])
    x[kind == 4, :19000] = -np.inf
    x[kind == 5, :] = -np.inf
    x[kind == 6, :] = low
    x[kind == 7, 777] = np.inf
    x[kind == 8, :] *= 1e30
    x[kind == 9, 1:] = np.nan
    check(x, rng.uniform(size=batch).astype(np.float32), NAMES, settings_of(rng, batch, vocab), dtype, 5, cuda)


def test_top_p_close_to_one_and_hot_and_cold(cuda):
    """What the one pass over a row bets on or bounds: shares near 1, temperatures far from 1, heavy and light tails."""
    rng = np.random.default_rng(22)
    batch, vocab = 640, 30000
    a = np.exp(rng.uniform(np.log(0.2), np.log(8.0), (batch, 1)))
    x = (5.0 - a * np.log(np.maximum(rng.uniform(size=(batch, vocab)), 2.0**-25) * vocab)).astype(np.float32)
    t = np.exp(rng.uniform(np.log(0.01), np.log(50.0), batch)).astype(np.float32)
    p = (1.0 - np.exp(rng.uniform(np.log(1e-6), np.log(0.9), batch))).astype(np.float32)
    check(x, rng.uniform(size=batch).astype(np.float32), ("temperature", "top_p"), (t, p), dev=cuda)
    # the largest ids of a vocabulary sorted by frequency come first, or last
    check(np.sort(x, 1)[:, ::-1].copy(), rng.uniform(size=batch).astype(np.float32), ("temperature", "top_p"), (t, p), dev=cuda)
    check(np.sort(x, 1), rng.uniform(size=batch).astype(np.float32), ("temperature", "top_p"), (t, p), dev=cuda)


@pytest.mark.parametrize("k", [1, 7, 256, 257, 1000, 1024, 1025, 5000])
def test_top_k_sizes(cuda, k):
    rng = np.random.default_rng(23)
    for batch in (3, 650):
        x = rows_of(rng, batch, 12000, "normal")
        check(x, rng.uniform(size=batch).astype(np.float32), ("top_k", "top_p"),
              (np.full(batch, k, np.int32), np.where(np.arange(batch) % 2, 0.9, 1.0).astype(np.float32)), dev=cuda)
