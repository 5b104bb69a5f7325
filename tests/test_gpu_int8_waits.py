"""Waits of the 8-bit product that run out (include/noel_sampler_cuda.h): the
call ends soon after the first of them, is reported, and leaves the next call
as it was."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

WAIT = -6
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


@pytest.mark.parametrize("tokens,cols", [(1, 2048), (17, 2048), (64, 2048), (128, 2048), (600, 2048),
                                         (1, 131_071), (64, 131_071), (128, 131_071), (600, 131_071)])
@pytest.mark.parametrize("limit", [1, 100_000])
def test_waits_that_run_out_while_copies_are_on_their_way(cuda, limits, tokens, cols, limit):
    """Limits in the range of a copy's latency, and of a tile's time where there are many columns (the results wait for
    a whole tile): whichever wait runs out first, the call is reported or right."""
    import torch

    from noel_b200 import sampler as S

    w, x = rows(30_000 if cols == 2048 else 3_000, cols, cuda, 3), rows(tokens, cols, cuda, 4)
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


def test_reports_go_to_their_streams(cuda, limits):
    """A check of one stream neither takes nor clears what another stream's product has to report."""
    import torch

    from noel_b200 import sampler as S

    w, x = rows(300, 256, cuda, 5), rows(4, 256, cuda, 6)
    torch.cuda.synchronize()
    good, bad, idle = (torch.cuda.Stream() for _ in range(3))
    S.int8_product(x, w, stream=good)
    assert [S.sync_check(s) for s in (good, bad, idle)] == [0, 0, 0]
    for _ in range(3):
        limits(2_000_000, stall_next_call=True)
        S.int8_product(x, w, stream=bad)
        limits(0)
        S.int8_product(x, w, stream=good)
        bad.synchronize()
        assert [S.sync_check(s) for s in (idle, good, torch.cuda.current_stream())] == [0, 0, 0]
        assert [S.sync_check(bad), S.sync_check(bad)] == [WAIT, 0]
    # twice before a check is one report
    for _ in range(2):
        limits(2_000_000, stall_next_call=True)
        S.int8_product(x, w, stream=bad)
    assert [S.sync_check(good), S.sync_check(bad), S.sync_check(bad)] == [0, WAIT, 0]


def test_reports_of_many_streams_and_threads(cuda):
    """Each thread's stalled product on a stream of its own is its own report."""
    import threading

    import torch

    from noel_b200 import sampler as S

    w, x = rows(300, 256, cuda, 7), rows(4, 256, cuda, 8)
    torch.cuda.synchronize()
    got = {}

    def work(n):
        stream = torch.cuda.Stream()
        seen = []
        for turn in range(6):
            stall = (n + turn) % 3 == 0
            S.set_wait_limit(2_000_000, stall_next_call=stall)  # of this thread
            S.int8_product(x, w, stream=stream)
            seen.append(S.sync_check(stream) == (WAIT if stall else 0))
        got[n] = seen

    threads = [threading.Thread(target=work, args=(n,)) for n in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got == {n: [True] * 6 for n in range(6)}


CAPTURED = """
import torch
from noel_b200 import sampler as S

dev = torch.device("cuda:0")
w, x = S.int8_cast(torch.randn(300, 256, device=dev)), S.int8_cast(torch.randn(4, 256, device=dev))
S.int8_product(x, w)
g = torch.cuda.CUDAGraph()
S.set_wait_limit(2_000_000, stall_next_call=True)
with torch.cuda.graph(g):
    S.int8_product(x, w)
S.set_wait_limit(0)
streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
assert [S.sync_check(s) for s in streams[:2]] == [0, 0]
for turn in range(2):
    g.replay()
    torch.cuda.synchronize()
    assert [S.sync_check(s) for s in streams] == [-6, -6, -6], turn
    assert [S.sync_check(s) for s in streams] == [0, 0, 0], turn
S.int8_product(x, w, stream=streams[1])
assert [S.sync_check(s) for s in streams] == [0, 0, 0]
"""


def in_a_process(text):
    r = subprocess.run([sys.executable, "-c", text], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_reports_of_a_replayed_graph(cuda):
    """It may run on any stream, so each stream's next check has it.  In a process of its own: streams that later tests make would
    be told as well."""
    in_a_process(CAPTURED)


FIRST = """
import threading
import torch
from noel_b200 import sampler as S

dev = torch.device("cuda:0")
q = torch.randint(-128, 128, (700, 256), dtype=torch.int8, device=dev)
w, xs = S.Int8Rows(q, torch.ones(700, device=dev)), [S.Int8Rows(q[:n], torch.ones(n, device=dev)) for n in (3, 20, 64, 128, 300, 5)]
wants = [(x.q.double() @ q.double().T).float() for x in xs]
torch.cuda.synchronize()
gate, got = threading.Barrier(len(xs)), {}

def work(n):
    stream = torch.cuda.Stream()
    gate.wait()
    y = S.int8_product(xs[n], w, stream=stream)
    got[n] = S.sync_check(stream) == 0 and torch.equal(y, wants[n])

threads = [threading.Thread(target=work, args=(n,)) for n in range(len(xs))]
for t in threads:
    t.start()
for t in threads:
    t.join()
assert got == {n: True for n in range(len(xs))}, got
"""


def test_first_products_of_many_threads(cuda):
    """What the library sets up on its first product is set up by several threads at once."""
    in_a_process(FIRST)
