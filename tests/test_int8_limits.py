"""What the 8-bit path refuses before anything of it runs, without a GPU: every
status below comes before the first CUDA call."""
import ctypes as C

import pytest

OK, INVALID, TOO_LARGE = 0, -1, -4
P = 1 << 20  # an address that is never dereferenced


@pytest.fixture(scope="module")
def lib():
    from noel_b200 import build, sampler

    build.build()
    return sampler.lib()


def head(lib, lora=None, adapter=P, process=None, batch=2, work=P, size=1 << 20, ldx=64):
    from noel_b200.sampler import RequestParamsStruct

    params = RequestParamsStruct()
    return lib.noel_lmhead_i8_sample(C.byref(params), P, 64, P, P, 0, ldx, batch, 64, 10, C.byref(lora) if lora else None, adapter,
                                     C.byref(process) if process else None, P, P, None, None, P, work, size, None)


def lora_struct(**fields):
    from noel_b200.sampler import LoraStruct

    return LoraStruct(**{**dict(d_a=P, lda=64, stride_a=64 * 4, d_b=P, ldb=4, stride_b=40, type=30, n_adapters=1, rank=4), **fields})


def mask_struct(**fields):
    from noel_b200.sampler import LogitsParamsStruct

    return LogitsParamsStruct(**{**dict(d_mask=P, mld=1, mask_rows=2), **fields})


@pytest.mark.parametrize("broken", [dict(adapter=None), dict(lora=dict(d_a=None)), dict(lora=dict(d_b=None)),
                                    dict(lora=dict(n_adapters=-1)), dict(process=dict(mask_rows=1)),
                                    dict(process=dict(mask_rows=-1)), dict(process=dict(mld=0))])
def test_head_refuses_before_it_runs(lib, broken):
    """What the adapters or the processing would refuse of the batch, when the projection would have run already."""
    lora = lora_struct(**broken.get("lora", {}))
    process = mask_struct(**broken.get("process", {}))
    assert head(lib, lora=lora, adapter=broken.get("adapter", P), process=process) == INVALID
    if "process" in broken:
        assert head(lib, process=process) == INVALID
    else:
        assert head(lib, lora=lora, adapter=broken.get("adapter", P)) == INVALID


def test_head_needs_the_adapters_scratch(lib):
    size = lib.noel_lora_workspace_bytes(40, 256)
    assert size > lib.noel_i8_linear_workspace_bytes(40, 64)
    lora = lora_struct(ldb=256, rank=256)
    assert head(lib, lora=lora, batch=40, size=size - 1) == INVALID
    assert lib.noel_lmhead_i8_workspace_bytes(40, 64, 10, 256) == size


MOST = 2**31 - 513  # tokens or rows of a product


def product(lib, tokens=0, rows=0):
    # one of the two is 0, so that what is not refused has nothing to do
    return lib.noel_i8_product(P, 16, P, tokens, P, 16, P, rows, 16, P, 0, max(rows, 1), None)


def test_product_sizes_that_its_tiles_would_pass(lib):
    """Steps of whole tiles from the last row on end below 2^31."""
    for n in (MOST + 1, 2**31 - 256, 2**31 - 1):
        assert product(lib, tokens=n) == TOO_LARGE and product(lib, rows=n) == TOO_LARGE, n
    assert product(lib, tokens=MOST) == OK and product(lib, rows=MOST) == OK


def test_linear_sizes_that_its_tiles_would_pass(lib):
    def linear(tokens=0, rows=0):
        size = lib.noel_i8_linear_workspace_bytes(tokens, 16)
        return lib.noel_i8_linear(P, 0, 16, tokens, P, 16, P, rows, 16, P, 0, max(rows, 1), P, size, None)

    assert linear(tokens=MOST + 1) == TOO_LARGE and linear(rows=MOST + 1) == TOO_LARGE
    assert linear(tokens=MOST) == OK and linear(rows=MOST) == OK
