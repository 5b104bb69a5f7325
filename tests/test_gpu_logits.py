"""noel_logits_process against its plain 64-bit form: penalties, biases and
masks on fp32 and bf16 rows; what no rule touches keeps its bits."""
import numpy as np
import pytest

from tests.request_ops import process_plain, same_bits, within

pytestmark = pytest.mark.gpu


def bits(x, dtype):
    """numpy array of the row values' bits, as the GPU holds them."""
    import torch

    return x.view(torch.int32 if dtype == "f32" else torch.int16).cpu().numpy()


def build(B, V, dtype, seed, pad=0, H=0, lens=True, bias=0, masks=0, density=0.5, v_begin=0, zipf=True, rows_of_mask=True):
    """Rows, parameters (numpy) and the logits tensor's wider storage."""
    import torch

    g = np.random.Generator(np.random.PCG64(seed))
    x = (3.0 * g.standard_normal((B, V + pad))).astype(np.float32)
    t = torch.from_numpy(x).to(torch.float32 if dtype == "f32" else torch.bfloat16)
    p = {}
    if H:
        ids = (np.exp(g.random((B, H)) * np.log(V + 1.0)) - 1).astype(np.int64) if zipf else g.integers(0, V, (B, H))
        ids = ids + v_begin
        odd = g.random((B, H)) < 0.05  # padding, ids of other columns, ids of no column
        ids = np.where(odd, g.choice([-1, -7, v_begin - 1, v_begin + V, 2**31 - 1, -2**31], (B, H)), ids)
        p["history"] = ids.astype(np.int32)
        if lens:
            n = g.integers(0, H + 1, B)
            n[0] = H + 5  # more than there is
            if B > 1:
                n[1] = -3
            if B > 2:
                n[2] = 0
            p["history_lens"] = n.astype(np.int32)
            p["prompt_lens"] = (g.integers(-1, H + 2, B)).astype(np.int32)
        p["repetition"] = (1.0 + 0.4 * g.random(B)).astype(np.float32)
        p["frequency"] = (0.5 * g.standard_normal(B)).astype(np.float32)
        p["presence"] = (0.5 * g.standard_normal(B)).astype(np.float32)
    if bias:
        ids = g.integers(0, max(1, min(V, 2 * bias)), (B, bias)) + v_begin  # several ids occur twice and more
        ids[:, ::7] = -1
        p["bias_ids"] = ids.astype(np.int32)
        p["bias"] = (2.0 * g.standard_normal((B, bias))).astype(np.float32)
    if masks:
        words = (v_begin + V + 31) // 32 + 1
        m = (g.random((masks, words, 32)) < density)
        m[0] = True
        if masks > 1:
            m[1] = False  # leaves nothing
        if masks > 2:
            m[2] = False
            m[2, (v_begin + V - 1) // 32, (v_begin + V - 1) % 32] = True  # the last id alone
        p["mask"] = (m.astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32)
        if rows_of_mask:
            r = g.integers(-1, masks + 1, B)
            r[: min(B, masks)] = np.arange(min(B, masks))
            p["mask_rows"] = r.astype(np.int32)
    return t, p


def params(S, dev, p, v_begin=0):
    import torch

    return S.LogitsParams(v_begin=v_begin, **{k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).to(dev)
                                              for k, v in p.items()})


def check(cuda, t, p, V, dtype, v_begin=0, run=None):
    from noel_b200 import sampler as S

    d = t.to(cuda)
    before = bits(d, dtype)
    want, bound, touched = process_plain(t[:, :V].double().numpy(), dtype=dtype, v_begin=v_begin, **p)
    prm = params(S, cuda, p, v_begin)
    if run is None:
        assert S.logits_process(d, prm, vocab=V) is d
    else:
        run(d, prm)
    after = bits(d, dtype)
    same = np.ones(after.shape, bool)
    same[:, :V] = ~touched
    same_bits(after, before, same)
    within(d[:, :V].double().cpu().numpy(), want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,V,pad", [(1, 1, 0), (1, 33, 0), (3, 31, 5), (5, 1000, 24), (2, 8192, 0), (4, 8193, 7),
                                     (3, 50001, 3), (40, 2049, 1)])
def test_process_everything_gpu(cuda, B, V, pad, dtype):
    t, p = build(B, V, dtype, seed=B * V + pad, pad=pad, H=100, bias=21, masks=min(B, 5))
    check(cuda, t, p, V, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("part", ["history", "history_all", "bias", "mask", "mask_each", "nothing"])
def test_process_one_part_gpu(cuda, part, dtype):
    kw = {"history": dict(H=70), "history_all": dict(H=70, lens=False, zipf=False), "bias": dict(bias=40),
          "mask": dict(masks=3), "mask_each": dict(masks=9, rows_of_mask=False), "nothing": {}}[part]
    t, p = build(9, 3001, dtype, seed=11, pad=2, **kw)
    check(cuda, t, p, 3001, dtype)


@pytest.mark.parametrize("without", ["repetition", "frequency", "presence", "prompt_lens", "history_lens"])
def test_process_parts_left_out_gpu(cuda, without):
    t, p = build(6, 700, "f32", seed=5, H=300)
    del p[without]
    check(cuda, t, p, 700, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H", [1, 31, 1023, 1024, 1025, 2047, 2048, 2049, 5000, 8192, 20000])
@pytest.mark.parametrize("bias", [0, 300])
def test_process_history_lengths_gpu(cuda, H, bias, dtype):
    t, p = build(4, 20011, dtype, seed=H, H=H, bias=bias, masks=2, density=0.9)
    check(cuda, t, p, 20011, dtype)


@pytest.mark.parametrize("bias", [1, 255, 256, 257, 3000, 16384])
def test_process_bias_lengths_gpu(cuda, bias):
    t, p = build(3, 9000, "f32", seed=bias, H=10, bias=bias)
    check(cuda, t, p, 9000, "f32")


def test_process_one_id_many_times_gpu(cuda):
    """a history and a bias list of one id only, and the sum in list order"""
    t, p = build(3, 500, "f32", seed=3, H=4000, bias=600)
    p["history"][:] = 17
    p["bias_ids"][:] = 17
    check(cuda, t, p, 500, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("density", [0.0, 0.003, 0.5, 0.99, 1.0])
@pytest.mark.parametrize("V", [64, 4096, 70003])
def test_process_mask_densities_gpu(cuda, V, density, dtype):
    t, p = build(7, V, dtype, seed=V, pad=3, masks=7, density=density)
    check(cuda, t, p, V, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v_begin", [1, 31, 32, 45, 100000])
def test_process_shards_gpu(cuda, v_begin, dtype):
    t, p = build(5, 9001, dtype, seed=v_begin, H=400, bias=30, masks=4, v_begin=v_begin)
    check(cuda, t, p, 9001, dtype, v_begin=v_begin)


def test_process_shards_give_the_whole_row_gpu(cuda):
    import torch

    from noel_b200 import sampler as S

    V, cuts = 10007, [0, 2501, 5001, 5002, 10007]
    t, p = build(6, V, "f32", seed=4, H=500, bias=50, masks=6)
    whole = S.logits_process(t.to(cuda), params(S, cuda, p))
    parts = t.to(cuda)
    for lo, hi in zip(cuts, cuts[1:]):
        S.logits_process(parts[:, lo:hi], params(S, cuda, p, v_begin=lo))
    assert torch.equal(whole, parts)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_process_special_values_gpu(cuda, dtype):
    """infinities, NaN and the types' extremes, untouched, penalised and masked"""
    import torch

    V = 4000
    t, p = build(5, V, dtype, seed=8, H=1500, bias=100, masks=5)
    g = np.random.Generator(np.random.PCG64(1))
    low = float(torch.finfo(t.dtype).min)
    v = torch.tensor([float("inf"), float("-inf"), float("nan"), low, 0.0, -0.0], dtype=t.dtype)
    t[:, torch.from_numpy(g.permutation(V)[:1200])] = v[torch.from_numpy(g.integers(0, 6, 1200))]
    p["bias"][:, :2] = np.inf
    check(cuda, t, p, V, dtype)


def test_process_keeps_nan_payloads_gpu(cuda):
    import torch

    from noel_b200 import sampler as S

    raw = torch.arange(0x7FC00000 + 1, 0x7FC00000 + 1 + 4 * 512, dtype=torch.int32).view(4, 512).to(cuda)
    x = raw.clone().view(torch.float32)
    h = torch.full((4, 3), 5, dtype=torch.int32, device=cuda)
    S.logits_process(x, S.LogitsParams(history=h, repetition=torch.full((4,), 2.0, device=cuda)))
    same = torch.ones(512, dtype=torch.bool, device=cuda)
    same[5] = False
    assert torch.equal(x.view(torch.int32)[:, same], raw[:, same])
    assert torch.isnan(x[:, 5]).all()


def test_process_misaligned_rows_gpu(cuda):
    """rows that start at any element, and buffers around them that stay as they were"""
    import torch

    from noel_b200 import sampler as S

    for dtype in ("f32", "bf16"):
        for off in (1, 2, 3):
            t, p = build(4, 2999, dtype, seed=off, H=64, bias=9, masks=4, density=0.3)
            store = torch.zeros(4 * 3005 + 8, dtype=t.dtype, device=cuda)
            view = store[off:off + 4 * 3005].view(4, 3005)[:, :2999]
            view.copy_(t)
            S.logits_process(view, params(S, cuda, p))
            want, bound, _ = process_plain(t.double().numpy(), dtype=dtype, **p)
            within(view.double().cpu().numpy(), want, bound)
            view.zero_()
            assert not store.any()


def test_process_strided_parameters_gpu(cuda):
    """histories, biases and masks in wider rows"""
    import torch

    from noel_b200 import sampler as S

    t, p = build(6, 900, "f32", seed=2, H=50, bias=12, masks=6)
    wide = {}
    for k, v in p.items():
        v = torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).to(cuda)
        if v.dim() == 2:
            w = torch.full((v.shape[0], v.shape[1] + 3), 1, dtype=v.dtype, device=cuda)
            w[:, :v.shape[1]] = v
            v = w[:, :v.shape[1]]
        wide[k] = v
    d = S.logits_process(t.to(cuda), S.LogitsParams(**wide))
    want, bound, _ = process_plain(t.double().numpy(), **p)
    within(d.double().cpu().numpy(), want, bound)


@pytest.mark.parametrize("B,V,H,masks", [(4, 5000, 200, 4), (3, 3000, 9000, 0)])
def test_process_in_a_graph_gpu(cuda, B, V, H, masks):
    """captured without a call before it, replayed on new values"""
    import torch

    def run(d, prm):
        g = torch.cuda.CUDAGraph()
        keep = d.clone()
        with torch.cuda.graph(g):
            from noel_b200 import sampler as S

            S.logits_process(d, prm)
        d.copy_(keep)
        g.replay()
        torch.cuda.synchronize()

    t, p = build(B, V, "f32", seed=9, H=H, bias=20, masks=masks)
    check(cuda, t, p, V, "f32", run=run)


def test_process_on_two_streams_gpu(cuda):
    import torch

    from noel_b200 import sampler as S

    t, p = build(16, 30000, "f32", seed=21, H=600, bias=20, masks=8)
    prm = params(S, cuda, p)
    want = S.logits_process(t.to(cuda), prm)
    streams = [torch.cuda.Stream() for _ in range(2)]
    rows = [t.to(cuda) for _ in range(8)]
    torch.cuda.synchronize()
    for i, d in enumerate(rows):
        S.logits_process(d, prm, stream=streams[i % 2])
    torch.cuda.synchronize()
    for d in rows:
        assert torch.equal(d, want)


@pytest.mark.parametrize("H,V", [(1000, 4096), (60000, 4096)])
def test_process_quotients_are_the_division_s_gpu(cuda, H, V):
    """x / repetition has the bits of the division, over all exponents and on
    both ways through (a table, and counted slices)"""
    import torch

    from noel_b200 import sampler as S

    g = torch.Generator(device=cuda).manual_seed(H)
    B = 64
    raw = torch.randint(0, 0x7F800000, (B, V), generator=g, device=cuda, dtype=torch.int32)  # every positive number
    raw[:, :64] = torch.randint(0x3F800000, 0x40000000, (B, 64), generator=g, device=cuda, dtype=torch.int32)
    x = raw.view(torch.float32)
    rep = torch.cat([1.0 + torch.rand(48, generator=g, device=cuda),
                     torch.tensor([1e-3, 2e-3, 0.3, 0.999, 1.0, 3.0, 1000.0, 1025.0, 1e9, 1e-9, 0.0, float("inf"), 1e38, 1e-38,
                                   1.5, 7.0], device=cuda)])
    h = torch.randint(0, V, (B, H), generator=g, device=cuda, dtype=torch.int32)
    seen = torch.zeros(B, V, dtype=torch.bool, device=cuda).scatter_(1, h.long(), True)
    want = torch.where(seen, x / rep[:, None], x)
    got = S.logits_process(x.clone(), S.LogitsParams(history=h, repetition=rep))
    same = (got.view(torch.int32) == want.view(torch.int32)) | (got.isnan() & want.isnan())
    assert same.all(), (x[~same][:5], got[~same][:5], want[~same][:5])


@pytest.mark.parametrize("H,bias", [(40, 8), (3000, 8), (9000, 0), (2000, 0)])
def test_process_large_batch_equals_small_ones_gpu(cuda, H, bias):
    """the ranges and kernels that a large batch takes give the bits that eight rows at a time give"""
    import torch

    from noel_b200 import sampler as S

    B, V = 1200, 50021
    g = torch.Generator(device=cuda).manual_seed(H)
    r = lambda *s: torch.rand(*s, generator=g, device=cuda)  # noqa: E731
    p = {"history": (torch.exp(r(B, H) * 10.8) - 1).to(torch.int32).clamp_(max=V - 1),
         "history_lens": torch.randint(0, H + 1, (B,), generator=g, device=cuda, dtype=torch.int32),
         "repetition": 1 + r(B), "frequency": r(B), "presence": r(B),
         "mask": torch.randint(-2**31, 2**31 - 1, (40, 1564), generator=g, device=cuda, dtype=torch.int32),
         "mask_rows": torch.randint(-1, 40, (B,), generator=g, device=cuda, dtype=torch.int32)}
    p["mask"][:10] = 0
    p["mask"][:10, 700] = 5
    p["mask"][10:20] = -1
    p["mask"][10:20, ::90] = -9
    if bias:
        p["bias_ids"] = torch.randint(0, V, (B, bias), generator=g, device=cuda, dtype=torch.int32)
        p["bias"] = r(B, bias)
    x = torch.randn(B, V, generator=g, device=cuda)
    got = S.logits_process(x.clone(), S.LogitsParams(**p))
    for b in range(0, B, 8):
        part = {k: v if k == "mask" else v[b:b + 8].contiguous() for k, v in p.items()}
        want = S.logits_process(x[b:b + 8].clone(), S.LogitsParams(**part))
        assert torch.equal(got[b:b + 8], want), b


def test_process_python_refusals_gpu(cuda):
    import torch

    from noel_b200 import sampler as S

    x = torch.zeros(2, 100, device=cuda)
    h = torch.zeros(3, 4, dtype=torch.int32, device=cuda)
    m = torch.zeros(2, 3, dtype=torch.int32, device=cuda)
    bad = [lambda: S.logits_process(x, S.LogitsParams(history=h)),                      # rows
           lambda: S.logits_process(x, S.LogitsParams(mask=m)),                         # words
           lambda: S.logits_process(x[:, ::2], S.LogitsParams()),                       # columns apart
           lambda: S.logits_process(x, S.LogitsParams(), vocab=101),
           lambda: S.logits_process(x.double(), S.LogitsParams()),
           lambda: S.LogitsParams(history=h.long()),
           lambda: S.LogitsParams(history=h, repetition=torch.ones(2, device=cuda)),
           lambda: S.LogitsParams(history=h, history_lens=torch.ones(3, dtype=torch.int32)),  # on the host
           lambda: S.LogitsParams(bias_ids=h, bias=torch.ones(3, 5, device=cuda)),
           lambda: S.logits_process(x, S.LogitsParams(history=h[:1].expand(2, 4)))]     # a pitch of 0
    for call in bad:
        with pytest.raises(S.NoelSamplerError):
            call()
    torch.cuda.synchronize()
    assert not x.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,H,bias,pad", [(60001, 9000, 0, 0), (60001, 9000, 300, 5), (152064, 9000, 300, 0),
                                          (152064, 1500, 21, 64), (24577, 30000, 16384, 31)])
@pytest.mark.parametrize("v_begin", [0, 45, 100000])
def test_process_long_histories_over_slices_gpu(cuda, v_begin, V, H, bias, pad, dtype):
    """several slices a row, rows on 32 bytes and off them, ids below and above a shard's columns"""
    t, p = build(4, V, dtype, seed=V + H + v_begin, pad=pad, H=H, bias=bias, masks=3, density=0.7, v_begin=v_begin)
    check(cuda, t, p, V, dtype, v_begin=v_begin)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_process_long_histories_uniform_and_whole_gpu(cuda, dtype):
    """ids of every line of every slice, all of them generated, no mask"""
    t, p = build(3, 100003, dtype, seed=8, pad=13, H=60000, lens=False, zipf=False)
    check(cuda, t, p, 100003, dtype)
