"""Plain 64-bit forms of the per-request operators (include/noel_logits.h,
include/noel_lora.h) and how far an fp32 computation may be from them.

Both bounds are sums of the roundings of a computation in fp32.  U is half a
step of fp32, 2^-24: one addition, product or quotient is off by at most
U |result|.  A matrix instruction aligns its products to the largest and cuts
them, so one of its steps is taken as off by at most 2 U of the sum of the
absolute products.
"""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 0.0, "bf16": 2.0 ** -8}  # of the last rounding, where the output has fewer bits
TINY = 2.0 ** -140


F32_MOST = float(np.finfo(np.float32).max)
BF16_OVER = 2.0 ** 128 - 2.0 ** 119  # half a step above bf16's largest value


def _f32_range(v):
    """v, or the infinity that an fp32 result of its size is"""
    return v if not abs(v) > F32_MOST else np.copysign(np.inf, v)


def process_plain(x, history=None, history_lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None,
                  bias_ids=None, bias=None, mask=None, mask_rows=None, v_begin=0, dtype="f32"):
    """(values, bound, touched) in float64 of numpy arrays; x [B, V] float64."""
    B, V = x.shape
    out, err = x.astype(np.float64).copy(), np.zeros((B, V))
    touched = np.zeros((B, V), bool)
    for b in range(B):
        if history is not None:
            H = history.shape[1]
            n = H if history_lens is None else min(max(int(history_lens[b]), 0), H)
            p = 0 if prompt_lens is None else int(prompt_lens[b])
            count, seen = {}, set()
            for i in range(n):
                c = int(history[b, i]) - v_begin
                if 0 <= c < V:
                    seen.add(c)
                    if i >= p:
                        count[c] = count.get(c, 0) + 1
            for c in seen:
                touched[b, c] = True
                v = out[b, c]
                if repetition is not None:
                    v = v / np.float64(repetition[b]) if v > 0 else v * np.float64(repetition[b])
                    v = _f32_range(v)
                    err[b, c] += U * abs(v)
                if c in count:
                    t = (np.float64(frequency[b]) if frequency is not None else 0.0) * count[c]
                    err[b, c] += U * (abs(t) + abs(v - t))
                    v = v - t - (np.float64(presence[b]) if presence is not None else 0.0)
                    v = _f32_range(v)
                    err[b, c] += U * abs(v)
                out[b, c] = v
        if bias_ids is not None:
            sums = {}
            for i, v in zip(bias_ids[b], bias[b]):
                c = int(i) - v_begin
                if 0 <= c < V:
                    sums.setdefault(c, []).append(np.float64(v))
            for c, vs in sums.items():
                touched[b, c] = True
                out[b, c] = _f32_range(out[b, c] + sum(vs))
                err[b, c] += U * ((len(vs) - 1) * sum(abs(v) for v in vs) + abs(out[b, c]))
        if mask is not None:
            m = b if mask_rows is None else int(mask_rows[b])
            if 0 <= m < mask.shape[0]:
                ids = v_begin + np.arange(V)
                ok = (mask[m].astype(np.uint32)[ids >> 5] >> (ids & 31).astype(np.uint32)) & 1
                out[b, ok == 0] = -np.inf
                err[b, ok == 0] = 0.0
                touched[b, ok == 0] = True
    if dtype == "bf16":
        over = touched & (np.abs(out) >= BF16_OVER)
        out[over] = np.copysign(np.inf, out[over])
    with np.errstate(invalid="ignore"):
        bound = 1.001 * err + HALF_STEP[dtype] * (np.abs(out) + err) + TINY
    return out, np.where(touched & np.isfinite(out), bound, 0.0), touched


def lora_plain(y, x, a, b, adapter, scale=None, ranks=None):
    """(values, bound) in float64; every argument a numpy array (a, b float64
    holding the adapters' own values).  The bound holds for cols up to 2048:
    no number of the first product goes through more than 96 additions, and
    none of the second through more than rank + 24."""
    out, bound = y.astype(np.float64).copy(), np.zeros(y.shape)
    for t, i in enumerate(adapter):
        if not 0 <= i < a.shape[0]:
            continue
        r = a.shape[1] if ranks is None else min(max(int(ranks[i]), 0), a.shape[1])
        A, Bm, xt = a[i, :r], b[i, :, :r], x[t].astype(np.float64)
        s = 1.0 if scale is None else np.float64(scale[i])
        low = s * (A @ xt)
        low_err = abs(s) * 96 * 2 * U * (np.abs(A) @ np.abs(xt)) + U * np.abs(low)
        out[t] += Bm @ low
        part = np.abs(Bm) @ (np.abs(low) + low_err)
        bound[t] = np.abs(Bm) @ low_err + (r + 24) * 2 * U * part + 2 * U * np.abs(out[t]) + TINY
    return out, 1.001 * bound


def same_bits(got, want, where):
    """got and want hold the same bits wherever where is set."""
    kind = {4: np.uint32, 2: np.uint16}[got.dtype.itemsize]
    np.testing.assert_array_equal(got.view(kind)[where], want.view(kind)[where])


def within(got, want, bound):
    """|got - want| <= bound where want is finite, and equal (NaN for NaN) where it is not."""
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    inf = ~fine & ~np.isnan(want)
    np.testing.assert_array_equal(got[inf], want[inf])
    with np.errstate(invalid="ignore"):
        off = np.where(fine, np.abs(got - want) - bound, 0.0)
    worst = np.unravel_index(np.argmax(off), off.shape)
    assert off[worst] <= 0, f"at {worst}: {got[worst]!r}, {want[worst]!r} +- {bound[worst]!r}"
