"""Batches of full-size rows of which the one pass settles few or none: wide
nuclei, large top-k, vocabularies sorted by frequency (include/noel_requests.h)."""
import numpy as np
import pytest

from tests.test_gpu_requests import check

pytestmark = pytest.mark.gpu

V = 152064


def normal(rng, batch, sd):
    return (rng.standard_normal((batch, V)) * sd).astype(np.float32)


def ranked(rng, batch, a):
    return (8.0 - a * np.log(np.maximum(rng.uniform(size=(batch, V)), 2.0**-25) * V)).astype(np.float32)


def uniforms(rng, batch):
    return rng.uniform(size=batch).astype(np.float32)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch", [1, 9, 80, 160])
def test_wide_nuclei(cuda, batch, dtype):
    rng = np.random.default_rng(31 + batch)
    p = rng.choice(np.array([0.8, 0.9, 0.95, 0.99], np.float32), batch)
    t = rng.choice(np.array([0.8, 1.0, 1.2], np.float32), batch)
    check(normal(rng, batch, 2.0), uniforms(rng, batch), ("temperature", "top_p"), (t, p), dtype, dev=cuda)
    check(ranked(rng, batch, 1.3), uniforms(rng, batch), ("temperature", "top_p"), (t, p), dtype, dev=cuda)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch", [5, 150])
def test_large_top_k(cuda, batch, dtype):
    rng = np.random.default_rng(41 + batch)
    k = rng.choice(np.array([1025, 2048, 2049, 30000, V - 1], np.int32), batch)
    p = rng.choice(np.array([0.5, 0.95, 1.0], np.float32), batch)
    check(normal(rng, batch, 3.0), uniforms(rng, batch), ("top_k", "top_p"), (k, p), dtype, dev=cuda)


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("batch", [3, 150])
def test_sorted_vocabularies(cuda, batch, rising):
    rng = np.random.default_rng(51 + batch)
    x = np.sort(ranked(rng, batch, rng.uniform(1.1, 2.5, (batch, 1)).astype(np.float32)), 1)
    x = x if rising else x[:, ::-1].copy()
    p = rng.choice(np.array([0.8, 0.9, 0.95], np.float32), batch)
    check(x, uniforms(rng, batch), ("top_p",), (p,), dev=cuda)
