"""Output weights in 8 bits to tokens on the GPU: noel_lmhead_i8_sample
against its steps called one by one and against their definitions, captured,
replayed on new inputs, and on two streams at once."""
import numpy as np
import pytest

from tests.request_sampling import sample_plain

pytestmark = pytest.mark.gpu


def setup(cuda, B, D, V, seed, adapters=True):
    import torch

    from noel_b200 import sampler as S

    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=cuda)

    s = {"w": S.int8_cast(randn(V, D) * D**-0.5 * 3), "x": randn(B, D), "u": torch.rand(B, generator=g, device=cuda)}
    s["params"] = S.SampleParams(temperature=torch.rand(B, generator=g, device=cuda) * 1.5,
                                 top_k=torch.randint(0, 60, (B,), generator=g, device=cuda, dtype=torch.int32) - 10,
                                 top_p=0.5 + 0.6 * torch.rand(B, generator=g, device=cuda),
                                 min_p=0.2 * torch.rand(B, generator=g, device=cuda) - 0.1)
    if adapters:
        s["adapters"] = S.Adapters((randn(3, 8, D) * D**-0.5).bfloat16(), randn(3, V, 8).bfloat16())
        s["adapter_ids"] = torch.randint(-1, 3, (B,), generator=g, device=cuda, dtype=torch.int32)
        history = torch.randint(0, V, (B, 20), generator=g, device=cuda, dtype=torch.int32)
        mask = torch.full((2, (V + 31) // 32), -1, dtype=torch.int32, device=cuda)
        mask[0, ::2] = 0
        mask[1] = 0
        rows = torch.full((B,), -1, dtype=torch.int32, device=cuda)
        rows[0] = 0
        rows[B // 2] = 1  # nothing is allowed
        s["process"] = S.LogitsParams(history=history, repetition=1 + torch.rand(B, generator=g, device=cuda), mask=mask, mask_rows=rows)
    return s


def steps(s, counts=True):
    from noel_b200 import sampler as S

    logits = S.int8_linear(s["x"], s["w"])
    if "adapters" in s:
        S.lora_apply(logits, s["x"], s["adapters"], s["adapter_ids"])
        S.logits_process(logits, s["process"])
    ids, probs, left = S.sample_requests(logits, s["u"], s["params"], counts=True)
    return ids, logits, probs, left


def whole(s):
    from noel_b200 import sampler as S

    return S.lmhead_int8_sample(s["w"], s["x"], s["u"], s["params"], adapters=s.get("adapters"),
                                adapter_ids=s.get("adapter_ids"), process=s.get("process"), counts=True)


def same(a, b):
    import torch

    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("B,D,V,adapters", [(1, 64, 1000, False), (5, 300, 32001, True), (70, 520, 5003, True),
                                            (300, 128, 2049, True)])
def test_path_is_its_steps(cuda, B, D, V, adapters):
    s = setup(cuda, B, D, V, B, adapters)
    out = whole(s)
    assert same(out, steps(s))
    p = s["params"].tensors
    ids, probs, counts = sample_plain(out[1].cpu().numpy(), s["u"].cpu().numpy(), *(t.cpu().numpy() for t in p))
    np.testing.assert_array_equal(out[0].cpu().numpy(), ids)
    np.testing.assert_array_equal(out[3].cpu().numpy(), counts)
    np.testing.assert_allclose(out[2].cpu().numpy(), probs, rtol=2.0**-23, atol=0)
    if adapters:
        assert out[0][B // 2] == -1 and counts[B // 2] == 0


def test_path_in_graphs_and_streams(cuda):
    import torch

    sets = [setup(cuda, B, 256, V, 7) for B, V in ((4, 30000), (200, 1500))]
    graphs, outs = [], []
    for s in sets:
        whole(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(whole(s))
        graphs.append(g)
    side = [torch.cuda.Stream() for _ in sets]
    for turn in range(3):
        for s in sets:
            s["x"].normal_()
            s["u"].uniform_()
        for stream, g in zip(side, graphs):  # both at once
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for s, out in zip(sets, outs):
            assert same(out, steps(s))


def test_refusals_leave_the_logits(cuda):
    """What a later step refuses is refused before the first one runs."""
    import torch

    from noel_b200 import sampler as S

    s = setup(cuda, 5, 64, 1000, 3)
    for broken in (dict(u=s["u"][:4]), dict(x=s["x"][:, :63]), dict(adapter_ids=None),
                   dict(process=S.LogitsParams(repetition=torch.ones(4, device=cuda))),
                   dict(params=S.SampleParams(temperature=torch.ones(4, device=cuda)))):
        with pytest.raises(S.NoelSamplerError):
            whole({**s, **broken})
    with pytest.raises(S.NoelSamplerError):
        whole({**s, "x": s["x"].bfloat16()})  # adapters want fp32
    assert same(whole(s), steps(s))


def test_empty_batches(cuda):
    import torch

    from noel_b200 import sampler as S

    w = S.int8_cast(torch.randn(100, 64, device=cuda))
    x, u = torch.empty(0, 64, device=cuda), torch.empty(0, device=cuda)
    assert S.int8_linear(x, w).shape == (0, 100) and S.int8_cast(x).q.shape == (0, 64)
    ids, logits, probs = S.lmhead_int8_sample(w, x, u, S.SampleParams())
    assert ids.numel() == probs.numel() == 0 and logits.shape == (0, 100)
    assert [t.numel() for t in S.sample_requests(logits, u, S.SampleParams(), counts=True)] == [0, 0, 0]
