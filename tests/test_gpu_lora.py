"""noel_lora_apply against its plain 64-bit form, element by element within
the bound of its own summation; rows without an adapter keep their bits."""
import numpy as np
import pytest

from tests.request_ops import lora_plain, same_bits, within

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]


def build(cuda, B, D, V, r, n, dtype, seed, pad=0, ragged=False, without=0.3, spoil=True):
    """Inputs on the GPU in wider rows (pad) whose padding is NaN, as are the
    ranks that an adapter does not use."""
    import torch

    g = np.random.Generator(np.random.PCG64(seed))
    tt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]

    def wide(x, t):
        w = torch.full(x.shape[:-1] + (x.shape[-1] + pad,), float("nan") if spoil else 0.0, dtype=t)
        w[..., :x.shape[-1]] = torch.from_numpy(x).to(t)
        return w.to(cuda)[..., :x.shape[-1]]

    f = lambda *s: g.standard_normal(s).astype(np.float32)  # noqa: E731
    s = {"y": wide(3 * f(B, V), torch.float32), "x": wide(f(B, D), torch.float32),
         "a": wide(f(n, r, D) * D ** -0.5, tt), "b": wide(f(n, V, r) * 0.5, tt),
         "scale": torch.from_numpy(0.5 + g.random(n).astype(np.float32)).to(cuda)}
    ids = g.integers(0, n, B)
    ids[g.random(B) < without] = -1
    if without and B > 3:
        ids[:3] = [n, 2**31 - 1, -2**31]
    s["ids"] = torch.from_numpy(ids.astype(np.int32)).to(cuda)
    s["ranks"] = None
    if ragged:
        ranks = g.integers(0, r + 1, n)
        ranks[0] = r + 3
        if n > 1:
            ranks[1] = -1
        s["ranks"] = torch.from_numpy(ranks.astype(np.int32)).to(cuda)
        for i, k in enumerate(ranks):
            if spoil:
                s["a"][i, max(k, 0):] = float("nan")
                s["b"][i, :, max(k, 0):] = float("nan")
    return s


def want(s):
    f = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    return lora_plain(f(s["y"]), f(s["x"]), f(s["a"]), f(s["b"]), s["ids"].cpu().numpy(), f(s["scale"]),
                      None if s["ranks"] is None else s["ranks"].cpu().numpy())


def apply(s, **kw):
    from noel_b200 import sampler as S

    ad = S.Adapters(s["a"], s["b"], scale=s["scale"], ranks=s["ranks"])
    assert S.lora_apply(s["y"], s["x"], ad, s["ids"], **kw) is s["y"]


def check(s):
    w, bound = want(s)
    whole = s["y"] if s["y"].is_contiguous() else s["y"].as_strided((s["y"].shape[0], s["y"].stride(0)), s["y"].stride())
    before = whole.cpu().numpy().copy()
    apply(s)
    after = whole.cpu().numpy()
    n = s["a"].shape[0]
    ids = s["ids"].cpu().numpy()
    keep = np.ones(after.shape, bool)
    keep[(ids >= 0) & (ids < n), :s["y"].shape[1]] = False
    same_bits(after, before, keep)
    within(s["y"].double().cpu().numpy(), w, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D,V,r,n", [
    (1, 1, 1, 1, 1), (1, 64, 1000, 16, 3), (2, 5, 31, 3, 2), (7, 1000, 4099, 12, 3), (16, 2048, 513, 16, 1),
    (17, 256, 777, 8, 1), (33, 96, 2000, 32, 2), (33, 97, 2001, 33, 4), (100, 512, 999, 64, 7), (64, 128, 640, 17, 64),
    (40, 72, 300, 128, 2), (9, 300, 1025, 256, 3), (130, 40, 130, 5, 2), (50, 128, 1000, 96, 2), (20, 64, 2052, 200, 2),
    (70, 64, 1004, 130, 3)])
def test_lora_gpu(cuda, B, D, V, r, n, dtype):
    check(build(cuda, B, D, V, r, n, dtype, seed=B + D + V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [1, 2, 8])
@pytest.mark.parametrize("r", [4, 16, 40])
def test_lora_wider_rows_gpu(cuda, r, pad, dtype):
    check(build(cuda, 21, 264, 1032, r, 3, dtype, seed=r + pad, pad=pad))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,pad", [(3, 13), (13, 3), (21, 11), (50, 14), (57, 7), (100, 4)])
def test_lora_odd_ranks_in_aligned_rows_gpu(cuda, r, pad, dtype):
    """rows of B on 16 bytes that end between two of them, NaN behind the rank"""
    check(build(cuda, 21, 256, 1060, r, 3, dtype, seed=r, pad=pad))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r", [8, 16, 48, 64, 128, 224])
def test_lora_ranks_of_their_own_gpu(cuda, r, dtype):
    check(build(cuda, 50, 200, 700, r, 6, dtype, seed=r, ragged=True))


@pytest.mark.parametrize("B", [255, 256, 257, 4095, 4097, 9000])
def test_lora_many_tokens_gpu(cuda, B):
    check(build(cuda, B, 64, 200, 8, 5, "bf16", seed=B))


def test_lora_one_adapter_for_all_gpu(cuda):
    check(build(cuda, 600, 128, 400, 16, 1, "bf16", seed=1, without=0.0))


def test_lora_more_adapters_than_tokens_gpu(cuda):
    check(build(cuda, 12, 128, 400, 16, 500, "f16", seed=1, without=0.0))


def test_lora_without_scale_and_without_any_adapter_gpu(cuda):
    s = build(cuda, 10, 128, 400, 16, 2, "bf16", seed=2)
    s["scale"] = None
    check(s)
    s = build(cuda, 10, 128, 400, 16, 2, "bf16", seed=3)
    s["ids"].fill_(-1)
    check(s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off", [1, 2, 3])
def test_lora_misaligned_gpu(cuda, off, dtype):
    """every array starting at an element of its own"""
    import torch

    s = build(cuda, 19, 136, 264, 16, 3, dtype, seed=off)
    for k in ("y", "x", "a", "b"):
        t = s[k].contiguous()
        store = torch.empty(t.numel() + 8, dtype=t.dtype, device=cuda)
        v = store[off:off + t.numel()].view(t.shape)
        v.copy_(t)
        s[k] = v
    check(s)


def test_lora_a_token_does_not_depend_on_the_others_gpu(cuda):
    import torch

    s = build(cuda, 90, 1000, 3001, 16, 4, "bf16", seed=6)
    y0 = s["y"].clone()
    apply(s)
    for rows in ([5], [0, 1, 2, 3, 4, 5, 6, 7], list(range(89, 20, -1))):
        at = torch.tensor(rows, device=cuda)
        part = {**s, "y": y0[at].clone(), "x": s["x"][at].contiguous(), "ids": s["ids"][at].contiguous()}
        apply(part)
        assert torch.equal(part["y"], s["y"][at])


@pytest.mark.parametrize("dtype,B,D,V,r,n", [("bf16", 300, 512, 40000, 64, 2), ("f16", 260, 1000, 30002, 16, 40),
                                             ("f32", 150, 777, 20001, 18, 3), ("bf16", 200, 640, 20003, 33, 3)])
def test_lora_large_equals_token_by_token_gpu(cuda, dtype, B, D, V, r, n):
    import torch

    s = build(cuda, B, D, V, r, n, dtype, seed=B, ragged=True)
    y0 = s["y"].clone()
    apply(s)
    for t in range(0, B, 37):
        part = {**s, "y": y0[t:t + 1].clone(), "x": s["x"][t:t + 1].contiguous(), "ids": s["ids"][t:t + 1].contiguous()}
        apply(part)
        assert torch.equal(part["y"].view(torch.int32), s["y"][t:t + 1].view(torch.int32)), t


def test_lora_special_values_stay_in_their_token_gpu(cuda):
    """infinities and NaN in one token's x reach that token's row only, and
    reach it as they do in the plain form"""
    import torch

    s = build(cuda, 20, 64, 300, 16, 1, "bf16", seed=7, without=0.0)
    s["x"][3, 5] = float("inf")
    s["x"][4, 6] = float("nan")
    s["a"][0, 2, 5] = 0.0
    clean = {**s, "y": s["y"].clone(), "x": torch.nan_to_num(s["x"], nan=0.0, posinf=0.0)}
    apply(s)
    apply(clean)
    rest = torch.tensor([t for t in range(20) if t not in (3, 4)], device=cuda)
    assert torch.equal(s["y"][rest], clean["y"][rest])
    assert torch.isnan(s["y"][3]).all() and torch.isnan(s["y"][4]).all()  # inf times the 0 of rank 2


def test_lora_infinite_product_gpu(cuda):
    """an infinity without a zero beside it stays an infinity"""
    import torch

    s = build(cuda, 3, 8, 40, 1, 1, "bf16", seed=7, without=0.0)
    s["a"].fill_(0.5)
    s["b"].copy_(torch.where(s["b"] > 0, 1.0, -1.0))
    s["x"][1, 2] = float("inf")
    sign = s["b"][0, :, 0] > 0
    apply(s)
    assert torch.equal(s["y"][1], torch.where(sign, float("inf"), float("-inf")))
    assert torch.isfinite(s["y"][0]).all() and torch.isfinite(s["y"][2]).all()


def test_lora_in_a_graph_gpu(cuda):
    """captured without a call before it, replayed on other adapter ids"""
    import torch

    from noel_b200 import sampler as S

    s = build(cuda, 24, 256, 900, 16, 3, "bf16", seed=12)
    ad = S.Adapters(s["a"], s["b"], scale=s["scale"])
    y0 = s["y"].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        S.lora_apply(s["y"], s["x"], ad, s["ids"])
    for shift in (0, 1, 2):
        s["ids"].copy_((s["ids"].clamp(min=-1, max=2) + shift) % 4 - 1)
        s["y"].copy_(y0)
        w, bound = want(s)
        g.replay()
        torch.cuda.synchronize()
        within(s["y"].double().cpu().numpy(), w, bound)


def test_lora_on_two_streams_gpu(cuda):
    import torch

    s = build(cuda, 40, 512, 5000, 16, 4, "bf16", seed=13)
    y0 = s["y"].clone()
    apply(s)
    streams = [torch.cuda.Stream() for _ in range(2)]
    copies = [{**s, "y": y0.clone()} for _ in range(8)]
    torch.cuda.synchronize()
    for i, c in enumerate(copies):
        apply(c, stream=streams[i % 2])
    torch.cuda.synchronize()
    for c in copies:
        assert torch.equal(c["y"], s["y"])


def test_lora_python_refusals_gpu(cuda):
    import torch

    from noel_b200 import sampler as S

    s = build(cuda, 4, 32, 64, 8, 2, "bf16", seed=1, pad=0)
    ad = S.Adapters(s["a"], s["b"])
    y0 = s["y"].clone()
    bad = [lambda: S.Adapters(s["a"], s["b"].float()), lambda: S.Adapters(s["a"], s["b"][:, :, :4]),
           lambda: S.Adapters(s["a"][:1], s["b"]), lambda: S.Adapters(s["a"][0], s["b"]),
           lambda: S.Adapters(s["a"], s["b"], scale=torch.ones(3, device=cuda)),
           lambda: S.Adapters(s["a"], s["b"], ranks=torch.ones(2, device=cuda)),
           lambda: S.lora_apply(s["y"][:, :60], s["x"], ad, s["ids"]),
           lambda: S.lora_apply(s["y"], s["x"][:3], ad, s["ids"]),
           lambda: S.lora_apply(s["y"], s["x"], ad, s["ids"].long()),
           lambda: S.lora_apply(s["y"], s["x"], ad, s["ids"].cpu()),
           lambda: S.lora_apply(s["y"][:1].expand(4, 64), s["x"], ad, s["ids"]),
           lambda: S.lora_apply(s["y"], s["x"].bfloat16(), ad, s["ids"])]
    for call in bad:
        with pytest.raises(S.NoelSamplerError):
            call()
    torch.cuda.synchronize()
    assert torch.equal(s["y"], y0)


def alone(s, y0, t):
    """token t's row of y where it is the whole batch"""
    part = {**s, "y": y0[t:t + 1].clone(), "x": s["x"][t:t + 1].contiguous(), "ids": s["ids"][t:t + 1].contiguous()}
    apply(part)
    return part["y"]


@pytest.mark.parametrize("dtype,B,D,V,r,n", [("bf16", 64, 4096, 300, 16, 64), ("bf16", 2048, 4096, 200, 64, 4),
                                             ("f16", 256, 4096, 264, 32, 8), ("f32", 150, 8192, 130, 33, 40),
                                             ("bf16", 2049, 2048, 130, 8, 2), ("f16", 2100, 5000, 77, 200, 3)])
def test_lora_a_token_alone_has_the_batch_s_bits_gpu(cuda, dtype, B, D, V, r, n):
    """columns enough for one token's to be shared by more CTAs than a batch's; the last tokens are a second pass's"""
    import torch

    s = build(cuda, B, D, V, r, n, dtype, seed=B + r, without=0.0)
    y0 = s["y"].clone()
    apply(s)
    for t in [*range(0, B, B // 8 + 1), B - 1]:
        assert torch.equal(alone(s, y0, t).view(torch.int32), s["y"][t:t + 1].view(torch.int32)), t


def test_lora_resident_adapters_change_no_bit_gpu(cuda):
    import torch

    s = build(cuda, 64, 4096, 300, 16, 256, "bf16", seed=21, without=0.0)
    s["ids"] %= 2
    few = {**s, "y": s["y"].clone(), "a": s["a"][:2], "b": s["b"][:2], "scale": s["scale"][:2]}
    apply(s)
    apply(few)
    assert torch.equal(few["y"].view(torch.int32), s["y"].view(torch.int32))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("r", [16, 24, 40, 64, 100, 128, 256])
def test_lora_the_layout_of_b_changes_no_bit_gpu(cuda, r, dtype):
    """rows of B on 16 bytes and on 2: the same sums in the same order"""
    import torch

    s = build(cuda, 40, 256, 1100, r, 3, dtype, seed=r, without=0.0)
    store = torch.zeros(3, 1100, r + 1 + r % 2, dtype=s["b"].dtype, device=cuda)
    store[:, :, :r] = s["b"]
    odd = {**s, "y": s["y"].clone(), "b": store[:, :, :r]}
    apply(s)
    apply(odd)
    assert torch.equal(odd["y"].view(torch.int32), s["y"].view(torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("r,far", [(128, 64), (128, 127), (200, 130), (256, 65), (256, 255)])
def test_lora_sums_of_64_ranks_are_added_in_fp32_gpu(cuda, r, far, pad, dtype):
    """Row v of B is 1 at rank 0 and c_v at a rank of another 64, A x is 1 at the one and 2^-23 at the other, y is 0: of the sum
    1 + c_v 2^-23, whose two numbers are exact, the fp32 addition's rounding is all that is left.  No c_v is a tie."""
    import torch

    c = torch.tensor([0.25, 0.375, 0.5625, 0.625, 0.75, 0.875, 0.9375, 1.25, 1.625, -0.125, -0.375, -0.75], device=cuda)
    V, tt = 12 * 31, {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    c = c.repeat(31)
    a = torch.zeros(1, r, 8, dtype=tt, device=cuda)
    a[0, 0, 0] = 1.0
    a[0, far, 1] = 1.0
    b = torch.zeros(1, V, r + pad, dtype=tt, device=cuda)
    b[0, :, 0] = 1.0
    b[0, :, far] = c
    x = torch.zeros(3, 8, device=cuda)
    x[:, 0], x[:, 1] = 1.0, 2.0 ** -23
    s = {"y": torch.zeros(3, V, device=cuda), "x": x, "a": a, "b": b[:, :, :r], "scale": None, "ranks": None,
         "ids": torch.zeros(3, dtype=torch.int32, device=cuda)}
    apply(s)
    assert torch.equal(s["y"], (1.0 + c.double() * 2.0 ** -23).float().expand(3, V))


@pytest.mark.parametrize("dtype", TYPES)
def test_lora_one_token_and_one_adapter_of_wider_rows_gpu(cuda, dtype):
    """a view of one token's row, and of one adapter, keeps the pitch that the rows have among others"""
    import torch

    s = build(cuda, 40, 1001, 301, 12, 3, dtype, seed=31, pad=7, without=0.0)
    s["ids"].fill_(1)
    y0 = s["y"].clone()
    apply(s)
    for t in (0, 7, 39):
        part = {**s, "y": y0[t:t + 1].clone(), "x": s["x"][t:t + 1], "a": s["a"][1:2], "b": s["b"][1:2],
                "scale": s["scale"][1:2], "ids": torch.zeros(1, dtype=torch.int32, device=cuda)}
        apply(part)
        assert torch.equal(part["y"].view(torch.int32), s["y"][t:t + 1].view(torch.int32)), t
