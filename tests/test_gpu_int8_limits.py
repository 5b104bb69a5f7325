"""The 8-bit path's refusals on the GPU: what is refused leaves every buffer as it was."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


def test_refused_batches_leave_their_buffers(cuda):
    """Adapters without ids and masks of fewer rows than the batch, through the C entry point."""
    import torch

    from noel_b200 import sampler as S

    B, D, V = 5, 64, 1000
    w = S.int8_cast(torch.randn(V, D, device=cuda))
    x, u = torch.randn(B, D, device=cuda), torch.rand(B, device=cuda)
    adapters = S.Adapters(torch.randn(2, 4, D, device=cuda).bfloat16(), torch.randn(2, V, 4, device=cuda).bfloat16())
    ids = torch.zeros(B, dtype=torch.int32, device=cuda)
    params = S.SampleParams()
    mask = torch.full((B, (V + 31) // 32), -1, dtype=torch.int32, device=cuda)
    process = S.LogitsParams(mask=mask)
    size = S.lib().noel_lmhead_i8_workspace_bytes(B, D, V, 4)
    work = torch.empty(size, dtype=torch.uint8, device=cuda)
    logits = torch.full((B, V), 7.0, device=cuda)
    drawn = torch.full((B,), 77, dtype=torch.int32, device=cuda)

    def call(lora=None, adapter=None, process=None):
        status = S.lib().noel_lmhead_i8_sample(
            params.ref, w.ptr, w.pitch, w.scale_ptr, x.data_ptr(), 0, D, B, D, V, lora, adapter, process, u.data_ptr(),
            drawn.data_ptr(), None, None, logits.data_ptr(), work.data_ptr(), size,
            C.c_void_p(torch.cuda.current_stream(cuda).cuda_stream))
        torch.cuda.synchronize()
        return status

    short = S.LogitsParamsStruct()
    C.memmove(C.byref(short), process.ref, C.sizeof(short))
    short.mask_rows = B - 1
    half = S.LoraStruct()
    C.memmove(C.byref(half), adapters.ref, C.sizeof(half))
    half.d_b = None
    for broken in (dict(lora=adapters.ref), dict(lora=C.byref(half), adapter=ids.data_ptr()), dict(process=C.byref(short)),
                   dict(lora=adapters.ref, adapter=ids.data_ptr(), process=C.byref(short))):
        assert call(**broken) == -1
        assert (logits == 7.0).all() and (drawn == 77).all()
    assert call(lora=adapters.ref, adapter=ids.data_ptr(), process=process.ref) == 0
    assert (logits != 7.0).all() and (drawn != 77).all()
