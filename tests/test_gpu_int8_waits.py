"""Waits of the 8-bit product that run out (include/noel_sampler_cuda.h): the
call ends soon after the first of them, is reported, and leaves the next call
as it was."""
import pytest

pytestmark = pytest.mark.gpu

WAIT = -6


@pytest.fixture
def limits():
    from noel_b200 import sampler as S

    yield S.set_wait_limit
    S.set_wait_limit(0)


def rows(n, cols, device, seed):
    import torch

    from noel_b200 import sampler as S

    return S.int8_cast(torch.randn(n, cols, generator=torch.Generator(device=device).manual_seed(seed), device=device))


@pytest.mark.parametrize("tokens", [4, 20, 64, 128, 600])
def test_a_stalled_product_of_many_tiles_ends_soon(cuda, limits, tokens):
    """Groups have 11 tiles (4 tokens, 1352 rows a CTA) to 31 (600): the limit holds for the call, not for each of them.
    What comes on top is the end's wait for what was issued, one millisecond, and the launch."""
    import torch

    from noel_b200 import sampler as S

    w, x = rows(200_000, 16, cuda, 1), rows(tokens, 16, cuda, 2)
    y = S.int8_product(x, w, dtype=torch.bfloat16)
    assert S.sync_check() == 0
    again = torch.empty_like(y)
    ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    limits(50_000_000, stall_next_call=True)
    ends[0].record()
    S.int8_product(x, w, out=again)
    ends[1].record()
    assert S.sync_check() == WAIT
    assert 45 <= ends[0].elapsed_time(ends[1]) < 110
    assert S.sync_check() == 0
    S.int8_product(x, w, out=again)
    assert S.sync_check() == 0
    assert torch.equal(again, y)


@pytest.mark.parametrize("tokens", [1, 17, 64, 128, 600])
@pytest.mark.parametrize("limit", [1, 3_000, 10_000, 30_000])
def test_waits_that_run_out_while_copies_are_on_their_way(cuda, limits, tokens, limit):
    """A limit in the range of a copy's latency: whichever wait runs out first, the call is reported or right."""
    import torch

    from noel_b200 import sampler as S

    w, x = rows(30_000, 2048, cuda, 3), rows(tokens, 2048, cuda, 4)
    y = S.int8_product(x, w)
    assert S.sync_check() == 0
    limits(limit)
    for _ in range(5):
        again = torch.empty_like(y)
        S.int8_product(x, w, out=again)
        status = S.sync_check()
        assert status in (0, WAIT)
        assert status == WAIT or torch.equal(again, y)
    limits(0)
    again = torch.empty_like(y)
    S.int8_product(x, w, out=again)
    assert S.sync_check() == 0
    assert torch.equal(again, y)
