"""The per-request operators without a GPU: their plain forms at known
answers, the C structs' layouts, the exported functions, and every refusal
(all of them come before the first CUDA call)."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from tests.request_ops import lora_plain, process_plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, TOO_LARGE, UNSUPPORTED = -1, -4, -5


@pytest.fixture(scope="module")
def lib():
    from noel_b200 import build, sampler

    build.build()
    return sampler.lib()


def test_process_plain_known_answers():
    x = np.array([[4.0, -2.0, 1.0, 0.5, 3.0, np.nan]])
    out, bound, touched = process_plain(
        x, history=np.array([[0, 1, 1, 2, 9, -1, 1]]), prompt_lens=np.array([2]), repetition=np.array([2.0]),
        frequency=np.array([0.25]), presence=np.array([0.5]), bias_ids=np.array([[3, 2, 3, -1]]),
        bias=np.array([[1.0, 2.0, 0.5, 9.0]]), mask=np.array([[0b001111]], np.uint32))
    # 0: prompt only; 1: 2 of 3 in the output; 2: once; 3: biased twice; 4, 5: masked
    np.testing.assert_array_equal(out, [[2.0, -4.0 - 0.5 - 0.5, 0.5 - 0.75 + 2.0, 2.0, -np.inf, -np.inf]])
    assert touched.all() and (bound < 1e-6).all()


def test_lora_plain_known_answers():
    a = np.array([[[1.0, 2.0], [0.0, 1.0]], [[3.0, 0.0], [7.0, 7.0]]])
    b = np.array([[[1.0, 1.0], [2.0, 0.0], [0.0, 1.0]], [[1.0, 9.0], [0.0, 9.0], [-1.0, 9.0]]])
    y = np.zeros((3, 3))
    out, _ = lora_plain(y, np.array([[1.0, 1.0], [2.0, 5.0], [1.0, 1.0]]), a, b, [0, 1, -1],
                        scale=np.array([1.0, 0.5]), ranks=np.array([2, 1]))
    np.testing.assert_array_equal(out, [[4.0, 6.0, 1.0], [3.0, 0.0, -3.0], [0.0, 0.0, 0.0]])


def test_headers_are_exported(lib):
    for header in ("noel_logits.h", "noel_lora.h", "noel_lmhead.h"):
        text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", header)).read(), flags=re.S)
        names = re.findall(r"^[A-Za-z_][\w \t\*]*?\b(noel_\w+)\s*\(", text, flags=re.M)
        assert names
        for name in names:
            assert hasattr(lib, name), name


def test_struct_layouts(tmp_path):
    """The ctypes structs have the C compiler's own offsets."""
    import subprocess

    from noel_b200.sampler import LogitsParamsStruct, LoraStruct

    lines = []
    for ctype, struct in (("noel_logits_params_t", LogitsParamsStruct), ("noel_lora_t", LoraStruct)):
        lines.append(f'printf("%zu\\n", sizeof({ctype}));')
        lines += [f'printf("%zu\\n", offsetof({ctype}, {name}));' for name, _ in struct._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "noel_logits.h"\n#include "noel_lora.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    want = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    have = []
    for struct in (LogitsParamsStruct, LoraStruct):
        have.append(C.sizeof(struct))
        have += [getattr(struct, name).offset for name, _ in struct._fields_]
    assert have == want


# addresses that are never dereferenced: the calls below are refused first
P, ODD = 1 << 20, (1 << 20) + 2


def _process(lib, batch=2, vocab=100, ld=100, dtype=0, logits=P, params=True, **kw):
    from noel_b200.sampler import LogitsParamsStruct

    s = LogitsParamsStruct(**kw)
    return lib.noel_logits_process(C.byref(s) if params else None, logits, dtype, batch, vocab, ld, None)


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(params=False)),
    (INVALID, dict(batch=-1)),
    (INVALID, dict(vocab=0)),
    (INVALID, dict(ld=99)),
    (INVALID, dict(dtype=7)),
    (INVALID, dict(logits=None)),
    (INVALID, dict(logits=ODD)),
    (INVALID, dict(logits=ODD + 1, dtype=1)),
    (INVALID, dict(v_begin=-1)),
    (INVALID, dict(v_begin=2**31 - 100)),
    (INVALID, dict(d_history=P, history_len=-1)),
    (INVALID, dict(d_history=P, history_len=5, hld=4)),
    (TOO_LARGE, dict(d_history=P, history_len=2**29, hld=2**29)),
    (INVALID, dict(d_history=ODD, history_len=5, hld=5)),
    (INVALID, dict(d_bias=P, bias_len=1, bld=1)),
    (INVALID, dict(d_bias_ids=P, bias_len=1, bld=1)),
    (INVALID, dict(d_bias_ids=P, d_bias=P, bias_len=-1)),
    (INVALID, dict(d_bias_ids=P, d_bias=P, bias_len=3, bld=2)),
    (TOO_LARGE, dict(d_bias_ids=P, d_bias=P, bias_len=16385, bld=16385)),
    (INVALID, dict(d_mask=P, mld=3, mask_rows=2)),
    (INVALID, dict(d_mask=P, mld=4, mask_rows=2, v_begin=29)),
    (INVALID, dict(d_mask=P, mld=4, mask_rows=1)),
    (INVALID, dict(d_mask=P, mld=4, mask_rows=-1, d_mask_rows=P)),
    (INVALID, dict(d_mask=ODD, mld=4, mask_rows=2)),
    (INVALID, dict(d_repetition=ODD)),
    (TOO_LARGE, dict(batch=2**31 - 1, vocab=2**20, ld=2**20)),
])
def test_process_refusals(lib, status, kw):
    assert _process(lib, **kw) == status
    assert lib.noel_sampler_cuda_last_error() == status
    assert lib.noel_sampler_cuda_last_error_message()


def test_process_of_no_rows_is_ok(lib):
    assert _process(lib, batch=0, logits=None) == 0


def _lora(lib, adapter=P, x=P, ldx=64, batch=3, cols=64, rows=50, y=P, ldy=50, work=P, work_bytes=None, lora=True, **kw):
    from noel_b200.sampler import LoraStruct

    s = LoraStruct(**{**dict(d_a=P, lda=64, stride_a=64 * 8, d_b=P, ldb=8, stride_b=50 * 8, type=30, n_adapters=2,
                             rank=8), **kw})
    need = lib.noel_lora_workspace_bytes(batch, s.rank) if work_bytes is None else work_bytes
    return lib.noel_lora_apply(C.byref(s) if lora else None, adapter, x, ldx, batch, cols, rows, y, ldy, work, need, None)


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(lora=False)),
    (UNSUPPORTED, dict(type=2)),
    (TOO_LARGE, dict(rank=0)),
    (TOO_LARGE, dict(rank=257, ldb=257)),
    (INVALID, dict(batch=-1)),
    (INVALID, dict(cols=0)),
    (INVALID, dict(rows=0)),
    (INVALID, dict(n_adapters=-1)),
    (INVALID, dict(ldx=63)),
    (INVALID, dict(ldy=49)),
    (INVALID, dict(lda=63)),
    (INVALID, dict(ldb=7)),
    (INVALID, dict(d_a=P + 1)),
    (INVALID, dict(d_b=ODD, type=0)),
    (INVALID, dict(d_a=None)),
    (INVALID, dict(d_b=None)),
    (INVALID, dict(adapter=None)),
    (INVALID, dict(adapter=ODD)),
    (INVALID, dict(x=None)),
    (INVALID, dict(x=ODD)),
    (INVALID, dict(y=None)),
    (INVALID, dict(y=ODD)),
    (INVALID, dict(d_scale=ODD)),
    (INVALID, dict(d_ranks=ODD)),
    (INVALID, dict(work=None)),
    (INVALID, dict(work=P + 4)),
    (INVALID, dict(work_bytes=3)),
])
def test_lora_refusals(lib, status, kw):
    assert _lora(lib, **kw) == status
    assert lib.noel_sampler_cuda_last_error() == status
    assert lib.noel_sampler_cuda_last_error_message()


def test_lora_of_nothing_is_ok(lib):
    assert _lora(lib, batch=0, x=None, y=None, adapter=None, work=None) == 0
    assert _lora(lib, n_adapters=0, d_a=None, d_b=None, work=None) == 0
    assert lib.noel_lora_workspace_bytes(0, 8) == 0


def test_lmhead_ex_refuses_before_the_projection(lib):
    from noel_b200.sampler import LogitsParamsStruct, LoraStruct, make_config

    def call(lora, process):
        return lib.noel_lmhead_sample_ex(
            C.byref(make_config()), P, 30, 64, P, 64, 2, 64, 50, C.byref(lora) if lora else None, P,
            C.byref(process) if process else None, None, 0, 0, P, P, None, P, P, 1 << 20, None)

    good = dict(d_a=P, lda=64, stride_a=512, d_b=P, ldb=8, stride_b=400, type=30, n_adapters=2, rank=8)
    assert call(LoraStruct(**{**good, "type": 5}), None) == UNSUPPORTED
    assert call(LoraStruct(**{**good, "lda": 8}), None) == INVALID
    assert call(None, LogitsParamsStruct(v_begin=-2)) == INVALID


def test_python_refusals_without_a_gpu():
    import torch

    from noel_b200 import sampler as S

    h = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(S.NoelSamplerError):
        S.LogitsParams(history=h)  # not on a GPU
    with pytest.raises(S.NoelSamplerError):
        S.LogitsParams(bias_ids=h)
    with pytest.raises(S.NoelSamplerError):
        S.LogitsParams(history_lens=h[:, 0])
    with pytest.raises(S.NoelSamplerError):
        S.LogitsParams(mask_rows=h[:, 0])
    with pytest.raises(S.NoelSamplerError):
        S.logits_process(torch.zeros(2, 8), S.LogitsParams())
    with pytest.raises(S.NoelSamplerError):
        S.logits_process(torch.zeros(2, 8, dtype=torch.float16), S.LogitsParams())
    with pytest.raises(S.NoelSamplerError):
        S.Adapters(torch.zeros(1, 2, 8), torch.zeros(1, 9, 2))
    with pytest.raises(S.NoelSamplerError):
        S.Adapters(torch.zeros(1, 2, 8, dtype=torch.int32), torch.zeros(1, 9, 2))


@pytest.mark.parametrize("v_begin", [-1, 2**31, 2**32, 2**32 + 5, -2**32 + 5])
def test_python_refuses_a_first_id_that_is_no_int(v_begin):
    """not taken for its lowest 32 bits"""
    from noel_b200 import sampler as S

    with pytest.raises(S.NoelSamplerError):
        S.LogitsParams(v_begin=v_begin)
