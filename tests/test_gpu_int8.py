"""8-bit projections on the GPU (include/noel_int8.h) against the definition:
casts against quotients in 64 bits, products bit for bit against whole-number
sums and the stated roundings."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FLOOR = np.float32(2.0**-126)


def cast_plain(x):
    """(q, scale) of the definition; x holds the input type's values."""
    x = x.astype(np.float32)
    top = np.abs(x).max(1)
    scale = np.maximum(top / np.float32(127), FLOOR)  # fp32 division
    bad = ~np.isfinite(top)
    # in 64 bits no quotient of two fp32 numbers is rounded onto a half: the two have 24 bits, a half of at most 8 more
    q = np.rint(np.where(bad[:, None], 0, x).astype(np.float64) / np.where(bad, 1, scale).astype(np.float64)[:, None])
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), scale)


def product_plain(a, a_scale, w, w_scale):
    total = (a.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32)  # whole numbers below 2^53, rounded once
    return (total * w_scale[None, :].astype(np.float32)) * a_scale[:, None].astype(np.float32)


def rows_i8(rng, rows, cols, device, pad=0):
    import torch

    pitch = (cols + 15) // 16 * 16 + 16 * pad
    full = torch.from_numpy(rng.integers(-128, 128, (rows, pitch), dtype=np.int8)).to(device)
    return full[:, :cols]


def same_bits(got, want):
    np.testing.assert_array_equal(got.view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols,pitch", [(1, 1, 1), (3, 15, 15), (5, 16, 16), (7, 1000, 1001), (2, 4096, 4096),
                                             (300, 129, 136), (1, 20011, 20011)])
def test_cast(cuda, dtype, rows, cols, pitch):
    import torch

    from noel_b200 import sampler as S

    rng = np.random.default_rng(rows * 7919 + cols)
    x = rng.standard_normal((rows, pitch)).astype(np.float32) * np.exp(rng.uniform(-8, 8, (rows, 1))).astype(np.float32)
    if rows > 2:
        x[2] = 0.0
    t = torch.from_numpy(x).to(cuda, getattr(torch, dtype))[:, :cols]
    out = S.int8_cast(t)
    q, scale = cast_plain(t.float().cpu().numpy())
    np.testing.assert_array_equal(out.q.cpu().numpy(), q)
    same_bits(out.scale.cpu().numpy(), scale)


def test_cast_ties_and_extremes(cuda):
    import torch

    from noel_b200 import sampler as S

    half = np.arange(-127, 127, dtype=np.float32) + 0.5
    near = np.nextafter(half, np.float32(200)), np.nextafter(half, np.float32(-200))
    tie = np.concatenate([half, *near, [127.0]]).astype(np.float32)  # the scale is exactly 1
    rows = [tie, tie * np.float32(2.0**100), tie * np.float32(2.0**-126), np.where(tie == 127, 127, tie / 3).astype(np.float32),
            np.full_like(tie, np.float32(3.4028235e38)), np.full_like(tie, np.float32(1.4e-45)),
            np.linspace(0, 5e-39, tie.size, dtype=np.float32), np.zeros_like(tie)]
    for bad in (np.nan, np.inf, -np.inf):
        r = tie.copy()
        r[5] = bad
        rows.append(r)
    x = np.stack(rows)
    out = S.int8_cast(torch.from_numpy(x).to(cuda))
    q, scale = cast_plain(x)
    np.testing.assert_array_equal(out.q.cpu().numpy(), q)
    np.testing.assert_array_equal(out.scale.cpu().numpy(), scale)
    assert np.isnan(out.scale.cpu().numpy()[-3:]).all()


@pytest.mark.parametrize("tokens,rows,cols", [
    (1, 1, 1), (1, 33, 16), (2, 500, 31), (1, 4096, 4096), (16, 129, 128), (17, 5000, 1000), (33, 257, 200),
    (64, 19001, 129), (65, 300, 64), (128, 128, 384), (129, 2049, 160), (256, 40000, 256), (257, 1025, 513),
    (700, 3000, 96), (1000, 77, 4000), (2049, 640, 48), (3, 20, 131071)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_product(cuda, tokens, rows, cols, dtype):
    import torch

    from noel_b200 import sampler as S

    rng = np.random.default_rng(tokens + 1000 * rows + cols)
    a, w = rows_i8(rng, tokens, cols, cuda), rows_i8(rng, rows, cols, cuda, pad=1)
    if cols > 100000:  # the largest sums
        a[0], w[0] = -128, -128
    sa = rng.uniform(0.001, 2, tokens).astype(np.float32)
    sw = rng.uniform(0.001, 2, rows).astype(np.float32)
    y = torch.full((tokens, rows + 3), 7.0, dtype=getattr(torch, dtype), device=cuda)
    got = S.int8_product(S.Int8Rows(a, torch.from_numpy(sa).to(cuda)), S.Int8Rows(w, torch.from_numpy(sw).to(cuda)),
                         out=y[:, :rows])
    assert S.sync_check() == 0
    want = torch.from_numpy(product_plain(a.cpu().numpy(), sa, w.cpu().numpy(), sw)).to(getattr(torch, dtype))
    assert torch.equal(got.cpu(), want)
    assert (y[:, rows:] == 7.0).all()


@pytest.mark.parametrize("tokens,rows,cols,dtype", [(1, 1000, 64, "bfloat16"), (23, 32001, 1000, "float32"),
                                                    (40, 500, 4096, "float16"), (300, 700, 1000, "bfloat16")])
def test_linear(cuda, tokens, rows, cols, dtype):
    import torch

    from noel_b200 import sampler as S

    rng = np.random.default_rng(tokens)
    x = torch.from_numpy(rng.standard_normal((tokens, cols)).astype(np.float32)).to(cuda, getattr(torch, dtype))
    x[tokens // 2] = 0.0
    w = S.int8_cast(torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32)).to(cuda))
    y = S.int8_linear(x, w)
    q, scale = cast_plain(x.float().cpu().numpy())
    same_bits(y.cpu().numpy(), product_plain(q, scale, w.q.cpu().numpy(), w.scale.cpu().numpy()))
    assert torch.equal(y, S.int8_product(S.int8_cast(x), w))


def test_linear_spoiled_token(cuda):
    """An infinity or a NaN spoils its token's results and no others."""
    import torch

    from noel_b200 import sampler as S

    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((20, 300)).astype(np.float32)).to(cuda)
    w = S.int8_cast(torch.from_numpy(rng.standard_normal((700, 300)).astype(np.float32)).to(cuda))
    clean = S.int8_linear(x, w)
    x[3, 7], x[9, 0] = float("inf"), float("nan")
    y = S.int8_linear(x, w)
    bad = torch.zeros(20, dtype=torch.bool)
    bad[[3, 9]] = True
    assert torch.isnan(y.cpu()[bad]).all()
    assert torch.equal(y.cpu()[~bad], clean.cpu()[~bad])


def test_results_do_not_depend_on_the_batch(cuda):
    import torch

    from noel_b200 import sampler as S

    rng = np.random.default_rng(6)
    x = torch.from_numpy(rng.standard_normal((600, 520)).astype(np.float32)).to(cuda)
    w = S.int8_cast(torch.from_numpy(rng.standard_normal((3001, 520)).astype(np.float32)).to(cuda))
    whole = S.int8_linear(x, w)
    for at, n in ((0, 1), (5, 16), (100, 31), (3, 64), (70, 100), (200, 256), (0, 300)):
        assert torch.equal(S.int8_linear(x[at:at + n], w), whole[at:at + n])


def test_stalled_product_is_reported(cuda):
    """A product whose loads never come gives up within its limit and is reported."""
    import torch

    from noel_b200 import sampler as S

    w = S.int8_cast(torch.randn(300, 256, device=cuda))
    x = S.int8_cast(torch.randn(300, 256, device=cuda))
    assert S.sync_check() == 0
    for tokens in (4, 300):
        a = S.Int8Rows(x.q[:tokens], x.scale[:tokens])
        try:
            S.set_wait_limit(2_000_000, stall_next_call=True)
            S.int8_product(a, w)
            assert S.sync_check() == -6
        finally:
            S.set_wait_limit(0)
        assert S.sync_check() == 0
        assert torch.isfinite(S.int8_product(a, w)).all()
        assert S.sync_check() == 0


def test_graph_and_streams(cuda):
    """Captured and replayed on new inputs, two graphs interleaved, and a stream other than the current one."""
    import torch

    from noel_b200 import sampler as S

    w = S.int8_cast(torch.randn(2000, 640, device=cuda))
    xs = [torch.randn(n, 640, device=cuda) for n in (5, 90)]
    graphs, outs = [], []
    for x in xs:
        S.int8_linear(x, w)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(S.int8_linear(x, w))
        graphs.append(g)
    for turn in range(3):
        for x in xs:
            x.normal_()
        for g in graphs:
            g.replay()
        for x, y in zip(xs, outs):
            assert torch.equal(y, S.int8_linear(x, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = S.int8_linear(xs[1], w, stream=side)
    side.synchronize()
    assert torch.equal(y, outs[1])
