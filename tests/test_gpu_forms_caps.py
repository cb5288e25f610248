"""GPU tests of capped scores whose tile holds scores beyond the cap that are no business of the row: at positions that it does not
see, or of other rows (qr_kv_attention_forms_dev), against the definition in 64 bits.

Tolerances (2-norm of a row, as in test_gpu_forms.py): a score z of a few nats far below its cap is off by a few steps of 32 bits of
itself, 10 x 2^-21 < 2^-17 of a nat and of a weight, which is inside what the roundings of the weights and the output leave.  A
score that is off by 2^-23 of the cap instead would be off by 0.1 at a cap of a million.
"""
import math

import pytest
import torch

from tests.chunkutil import TORCH, randn, row_errors
from tests.formutil import filled_as, forms64
from tests.test_gpu_forms import tol

pytestmark = pytest.mark.gpu

# (A score's size against its cap, and so which arithmetic a cap gets, goes by the scale: queries of 1 / scale leave the scores as they are.)
SCALES = [1.0, 64.0]
TYPES = [("bf16", "bf16"), ("f16", "f16"), ("e4m3", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("e4m3", "f16")]


@pytest.mark.parametrize("dtype,act", TYPES)
@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("n", [1, 12, 40, 150])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("odd", ["large", "inf", "nan"])
def test_keys_that_no_row_sees(gpu, odd, scale, n, D, dtype, act):
    """Keys in front of the first visible position, in its tile."""
    first, length = 293, 600
    x = {"large": 3e4 if dtype == "f16" else 1e30, "inf": math.inf, "nan": math.nan}[odd]

    def edit(i, k, v):
        for t in (256, 289, 291, 292):
            k[t] = x if t % 2 else -x

    kv, rows = filled_as(8, 2, D, dtype, [length], edit=edit)
    k, v = rows[0]
    k = k.clone()
    k[:first] = 0
    q = randn(3, n, 8, D, dtype=act, scale=1.6 / (scale * math.sqrt(D)))
    with kv:
        for cap in (30.0, 1e4, 1e5, 1e6):
            out = torch.empty(n, 8 * D, dtype=TORCH[act], device="cuda")
            kv.AttentionFormsDev(0, [0], [310], [n], q, out, scale, cap=cap, first=[first])
            want, size = forms64(q, k[:310 + n], v[:310 + n], 310, scale, 8, 2, cap=cap, first=first)
            e = row_errors(out.view(n, 8, D), want, size)
            assert e <= tol(dtype, act, cap), f"cap {cap}: {e:.3g}"


@pytest.mark.parametrize("dtype,act", TYPES)
@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("n", [1, 12, 40, 150])
@pytest.mark.parametrize("scale", SCALES)
def test_rows_beside_one_of_large_scores(gpu, scale, n, D, dtype, act):
    """One (query, head) row whose scores pass every cap, among rows of ordinary ones."""
    heads, length = 8, 500
    kv, rows = filled_as(heads, 2, D, dtype, [length])
    k, v = rows[0]
    q = randn(3, n, heads, D, dtype="f32", scale=1.6 / (scale * math.sqrt(D)))  # ordinary scores: 1.6 N(0, 1)
    q[n // 2, 1] = 4e4 / scale * torch.sign(q[n // 2, 1])
    q = q.to(TORCH[act])
    others = torch.ones(n, heads, dtype=torch.bool, device="cuda")
    others[n // 2, 1] = False
    with kv:
        for cap in (30.0, 1e4, 1e5, 6e5):
            z = scale * q[n // 2, 1].double() @ k[:length - n, 0].double().t().contiguous()
            assert z.abs().max() > cap / 2
            out = torch.empty(n, heads * D, dtype=TORCH[act], device="cuda")
            kv.AttentionFormsDev(0, [0], [length - n], [n], q, out, scale, cap=cap)
            want, size = forms64(q, k, v, length - n, scale, heads, 2, cap=cap)
            assert torch.isfinite(out).all()
            e = row_errors(out.view(n, heads, D)[others], want[others], size[others])
            assert e <= tol(dtype, act, cap), f"cap {cap}: {e:.3g}"
