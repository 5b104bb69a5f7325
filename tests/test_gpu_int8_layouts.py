"""8-bit projections of tokens whose rows are parts of wider ones, start
anywhere and go into parts of wider results, bit for bit."""
import numpy as np
import pytest

from tests.test_gpu_int8 import cast_plain, product_plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("tokens,rows,cols,first,wide,at,gap", [
    (1, 33, 17, 1, 2, 1, 4), (3, 500, 130, 3, 64, 5, 0), (17, 129, 1000, 1, 1, 0, 3), (40, 257, 96, 8, 24, 16, 16),
    (65, 300, 511, 0, 1, 7, 2), (130, 1025, 64, 5, 0, 1, 1), (300, 258, 200, 2, 7, 3, 9)])
def test_linear_of_parts(cuda, dtype, out, tokens, rows, cols, first, wide, at, gap):
    """Columns first .. first + cols of rows that are wide longer; results from column at on, gap columns behind them."""
    import torch

    from noel_b200 import sampler as S

    rng = np.random.default_rng(tokens * 31 + cols)
    full = torch.from_numpy(rng.standard_normal((tokens, first + cols + wide)).astype(np.float32)).to(cuda, getattr(torch, dtype))
    full[:, :first] = 1e4  # what lies beside a row does not count
    full[:, first + cols:] = float("nan")
    x = full[:, first:first + cols]
    w = S.int8_cast(torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32)).to(cuda))
    whole = torch.full((tokens + 1, at + rows + gap), 7.0, dtype=getattr(torch, out), device=cuda)
    y = whole[:tokens, at:at + rows]
    assert S.int8_linear(x, w, out=y) is y
    q, scale = cast_plain(x.float().cpu().numpy())
    want = torch.from_numpy(product_plain(q, scale, w.q.cpu().numpy(), w.scale.cpu().numpy())).to(getattr(torch, out))
    assert torch.equal(y.cpu(), want)
    whole[:tokens, at:at + rows] = 7.0
    assert (whole == 7.0).all()
    cast = S.int8_cast(x)
    assert torch.equal(S.int8_product(cast, w, dtype=getattr(torch, out)).cpu(), want)
