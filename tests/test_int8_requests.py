"""8-bit projections and sampling with every row's own settings, without a
GPU: the plain sampler at known answers, the C struct's layout, the exported
functions, and every refusal (all of them come before the first CUDA call)."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from tests.request_sampling import sample_plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, TOO_LARGE, UNSUPPORTED = -1, -4, -5
OK = 0

# addresses that are never dereferenced: the calls below are refused first, or have nothing to do
P, ODD = 1 << 20, (1 << 20) + 1


@pytest.fixture(scope="module")
def lib():
    from noel_b200 import build, sampler

    build.build()
    return sampler.lib()


def test_headers_are_exported(lib):
    for header in ("noel_int8.h", "noel_requests.h", "noel_lmhead.h"):
        text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", header)).read(), flags=re.S)
        names = re.findall(r"^[A-Za-z_][\w \t\*]*?\b(noel_\w+)\s*\(", text, flags=re.M)
        assert names
        for name in names:
            assert hasattr(lib, name), name


def test_struct_layout(tmp_path):
    import subprocess

    from noel_b200.sampler import RequestParamsStruct

    fields = [name for name, _ in RequestParamsStruct._fields_]
    lines = ['printf("%zu\\n", sizeof(noel_request_params_t));']
    lines += [f'printf("%zu\\n", offsetof(noel_request_params_t, {name}));' for name in fields]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "noel_requests.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    want = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert [C.sizeof(RequestParamsStruct)] + [getattr(RequestParamsStruct, n).offset for n in fields] == want


def test_sample_plain_known_answers():
    # weights 1, 2, 4, 8 of 15 at temperature 1; u goes by running sums in the order of ids
    x = np.log(np.array([1.0, 2.0, 4.0, 8.0]))
    for u, want in ((0.0, 0), (0.9 / 15, 0), (1.1 / 15, 1), (2.9 / 15, 1), (3.1 / 15, 2), (7.1 / 15, 3), (0.999, 3)):
        ids, probs, counts = sample_plain(x[None], [u])
        assert ids[0] == want and counts[0] == 4
        np.testing.assert_allclose(probs[0], 2.0**want / 15, rtol=1e-12)
    one = np.ones(1)
    # top-k 2: 4 and 8 of 12
    assert sample_plain(x[None], [0.32], top_k=one * 2)[0][0] == 2 and sample_plain(x[None], [0.34], top_k=one * 2)[0][0] == 3
    # top-p 0.7: 8 is less than 10.5, 8 + 4 is not; 0.53: 8 alone
    assert sample_plain(x[None], [0.5], top_p=one * 0.7)[2][0] == 2 and sample_plain(x[None], [0.5], top_p=one * 0.53)[2][0] == 1
    # top-p after top-k: 8 of 12 is 0.67
    assert sample_plain(x[None], [0.5], top_k=one * 2, top_p=one * 0.66)[2][0] == 1
    # min-p goes by the largest: 0.4 keeps 4 and 8
    assert sample_plain(x[None], [0.5], min_p=one * 0.4)[2][0] == 2
    # temperature 0.5 squares the weights: 64 of 85
    np.testing.assert_allclose(sample_plain(x[None], [0.9], temperature=one * 0.5)[1][0], 64 / 85, rtol=1e-12)
    # ties: the lower ids come first
    tie = np.zeros((1, 5))
    assert sample_plain(tie, [0.99], top_k=one * 2)[0][0] == 1 and sample_plain(tie, [0.0], temperature=one * 0)[0][0] == 0
    # nothing to draw
    assert sample_plain(np.full((1, 3), -np.inf), [0.5])[0][0] == -1


def cast(lib, x=P, kind=0, ldx=64, rows=2, cols=64, q=P, ldq=64, scale=P):
    return lib.noel_i8_cast(x, kind, ldx, rows, cols, q, ldq, scale, None)


def test_cast_refusals(lib):
    assert cast(lib, kind=2) == UNSUPPORTED
    assert cast(lib, cols=131072, ldx=131072, ldq=131072) == TOO_LARGE
    for bad in (dict(rows=-1), dict(cols=0), dict(ldx=63), dict(ldq=48), dict(ldq=72), dict(x=ODD), dict(q=P + 8),
                dict(scale=P + 2), dict(x=None), dict(q=None), dict(scale=None)):
        assert cast(lib, **bad) == INVALID, bad
    assert cast(lib, rows=0, x=None, q=None, scale=None) == OK
    assert lib.noel_sampler_cuda_last_error_message() == b""


def product(lib, a=P, lda=64, sa=P, tokens=2, w=P, ldw=64, sw=P, rows=3, cols=64, y=P, dtype=0, ldy=3):
    return lib.noel_i8_product(a, lda, sa, tokens, w, ldw, sw, rows, cols, y, dtype, ldy, None)


def test_product_refusals(lib):
    assert product(lib, dtype=2) == UNSUPPORTED
    assert product(lib, cols=131072, lda=131072, ldw=131072) == TOO_LARGE
    assert product(lib, lda=1 << 40) == TOO_LARGE
    for bad in (dict(tokens=-1), dict(rows=-1), dict(cols=0), dict(lda=48), dict(lda=72), dict(ldw=48), dict(ldw=72),
                dict(ldy=2), dict(a=P + 8), dict(w=P + 8), dict(sa=P + 1), dict(sw=P + 1), dict(y=P + 2), dict(a=None),
                dict(sa=None), dict(w=None), dict(sw=None), dict(y=None)):
        assert product(lib, **bad) == INVALID, bad
    assert product(lib, dtype=1, y=ODD) == INVALID
    assert product(lib, tokens=0, a=None, y=None) == OK and product(lib, rows=0, w=None, y=None) == OK


def test_linear_refusals(lib):
    def linear(x=P, kind=0, ldx=60, tokens=2, w=P, ldw=64, sw=P, rows=3, cols=60, y=P, dtype=0, ldy=3, work=P, size=1 << 20):
        return lib.noel_i8_linear(x, kind, ldx, tokens, w, ldw, sw, rows, cols, y, dtype, ldy, work, size, None)

    need = lib.noel_i8_linear_workspace_bytes(2, 60)
    assert need == 2 * (64 + 4) and lib.noel_i8_linear_workspace_bytes(0, 60) == 0
    for bad in (dict(work=None), dict(size=need - 1), dict(work=P + 8), dict(ldx=59), dict(ldw=56), dict(tokens=-1), dict(x=None),
                dict(w=None), dict(y=None)):
        assert linear(**bad) == INVALID, bad
    assert linear(kind=7) == UNSUPPORTED and linear(dtype=7) == UNSUPPORTED
    assert linear(cols=131072, ldx=131072, ldw=131072) == TOO_LARGE
    assert linear(tokens=0, x=None, work=None, size=0) == OK


def requests(lib, params="given", logits=P, dtype=0, batch=2, vocab=10, ld=10, u=P, ids=P, probs=P, counts=P, work=P, size=8, **fields):
    from noel_b200.sampler import RequestParamsStruct

    p = RequestParamsStruct(**fields)
    return lib.noel_sample_requests(C.byref(p) if params else None, logits, dtype, batch, vocab, ld, u, ids, probs, counts, work,
                                    size, None)


def test_request_refusals(lib):
    assert lib.noel_sample_requests_workspace_bytes(2, 10) == 8
    assert requests(lib, dtype=2) == UNSUPPORTED
    assert requests(lib, vocab=1048577, ld=1048577) == TOO_LARGE and requests(lib, batch=(1 << 24) + 1, size=1 << 30) == TOO_LARGE
    for bad in (dict(params=None), dict(batch=-1), dict(vocab=0), dict(ld=9), dict(logits=P + 2), dict(u=P + 2), dict(ids=P + 2),
                dict(probs=P + 2), dict(counts=P + 2), dict(work=P + 4), dict(work=None), dict(size=7), dict(logits=None),
                dict(u=None), dict(ids=None), dict(d_temperature=P + 1), dict(d_top_k=P + 2), dict(d_top_p=P + 2),
                dict(d_min_p=P + 3)):
        assert requests(lib, **bad) == INVALID, bad
    assert requests(lib, dtype=1, logits=ODD) == INVALID
    assert requests(lib, batch=0, logits=None, u=None, ids=None, work=None, size=0) == OK


def test_head_refusals(lib):
    from noel_b200.sampler import LoraStruct, RequestParamsStruct

    p = RequestParamsStruct()

    def head(params=p, w=P, ldw=64, sw=P, x=P, kind=0, ldx=64, batch=2, dim=64, vocab=10, lora=None, adapter=P, process=None, u=P,
             ids=P, logits=P, work=P, size=1 << 20):
        return lib.noel_lmhead_i8_sample(C.byref(params) if params else None, w, ldw, sw, x, kind, ldx, batch, dim, vocab,
                                         C.byref(lora) if lora else None, adapter, process, u, ids, None, None, logits, work, size,
                                         None)

    need = lib.noel_lmhead_i8_workspace_bytes(2, 64, 10, 0)
    assert need == lib.noel_i8_linear_workspace_bytes(2, 64)
    for bad in (dict(params=None), dict(w=None), dict(ldw=72), dict(x=None), dict(u=None), dict(ids=None), dict(logits=None),
                dict(work=None), dict(size=need - 1), dict(batch=-1), dict(vocab=0), dict(dim=0), dict(ldx=63)):
        assert head(**bad) == INVALID, bad
    lora = LoraStruct(d_a=P, lda=64, stride_a=64 * 4, d_b=P, ldb=4, stride_b=40, type=30, n_adapters=1, rank=4)
    assert head(lora=lora, kind=30) == UNSUPPORTED
    lora.rank = 257
    assert head(lora=lora) == TOO_LARGE
    lora.rank, lora.type = 4, 5
    assert head(lora=lora) == UNSUPPORTED
    assert head(batch=0, x=None, u=None, ids=None, logits=None, work=None, size=0) == OK


def test_python_refusals():
    import torch

    from noel_b200 import sampler as S

    x = torch.zeros(2, 32)
    for call in (lambda: S.int8_cast(x), lambda: S.Int8Rows(x.to(torch.int8), torch.zeros(2)),
                 lambda: S.SampleParams(temperature=torch.zeros(2)), lambda: S.SampleParams(top_k=torch.zeros(2)),
                 lambda: S.sample_requests(x, torch.zeros(2), S.SampleParams()),
                 lambda: S.sample_requests(x.half(), torch.zeros(2), S.SampleParams())):
        with pytest.raises(S.NoelSamplerError) as e:
            call()
        assert e.value.status == INVALID
