"""The softmax weights of the attention over the paged cache in its second
product, against float64: their rounding is well below a bf16 output's own,
whichever scales V has and however small they are."""
from __future__ import annotations

import numpy as np
import pytest

import cache_rows as R
from cache_plans import plan
from test_gpu_cache import Pool, draw16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t,out_t", [("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("way", list(R.WAYS))
def test_weights_of_every_kernel(torch_gpu, way, d, t, out_t):
    rng = np.random.default_rng(d)
    p = R.batch(torch_gpu, way, d)
    R.spread(p, rng)
    q, qv = R.queries(torch_gpu, rng, p, t)
    R.check(torch_gpu, p, q, qv, out_t)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shift", ["low", "high", "late", "last", "mixed"])
@pytest.mark.parametrize("way", list(R.WAYS))
def test_scales_of_v_past_fp16(torch_gpu, way, d, shift):
    """Values that fp16 does not hold, in one block of channels: from the first token on (2^-40, 2^95), from a token in
    the middle on, in the last visible token alone, and here and there beside blocks of zeros and of NaN."""
    rng = np.random.default_rng(d)
    p = R.batch(torch_gpu, way, d)
    first_block = np.arange(d // 32) == 0
    if shift in ("low", "high"):
        R.spread(p, rng, first_block * (-40 if shift == "low" else 95))
    else:
        R.spread(p, rng)
        _, _, page, _, _ = R.WAYS[way]
        for b, n in enumerate(p.lengths):
            slots = {"late": range(n // 2, n), "last": range(max(n - 1, 0), n),
                     "mixed": sorted(rng.integers(0, n, n // 40 + 1))}[shift] if n else ()
            for i, slot in enumerate(slots):
                at = p.table[b, slot // page], slice(None), slot % page, 0
                kind = i % 4 if shift == "mixed" else 0
                if kind < 2:
                    p.host["v_scales"][at] = (90, 141)[kind]
                elif kind == 2:
                    p.host["v_scales"][at] = 1
                    p.host["v_codes"][at[:3] + (slice(0, 16),)] = rng.integers(0, 2, 16) * 0x80  # zeros of both signs
                else:
                    p.host["v_scales"][at] = 255
        p.upload()
    q, qv = R.queries(torch_gpu, rng, p, "bf16")
    R.check(torch_gpu, p, q, qv, "bf16")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,most,kind", [(1, 1, "shares"), (70, 70, "splits"), (70, 33000, "chunk")])
@pytest.mark.parametrize("first", [True, False])
def test_many_small_weights(torch_gpu, d, new, most, kind, first):
    """One token of weight 1 without a value, first or last, and 20000 of 2^-22 with one: their sum is the output."""
    n = 20000
    p = Pool(torch_gpu, d, [0, new], [n], 1, 256, 1, seed=1, max_new=most)
    assert plan(p.shape, d).kind == kind
    for side in "kv":
        p.host[side + "_codes"][:] = 0
        p.host[side + "_scales"][:] = 127
    p.host["v_codes"][:] = 0x22  # 1.0
    slot = 0 if first else n - new  # seen by every row
    at = p.table[0, slot // 256], 0, slot % 256
    p.host["k_codes"][at + (0,)] = 6  # 4.0 in channel 0
    p.host["v_codes"][at] = 0
    p.upload()
    q = torch_gpu.zeros(1, new, 1, d, dtype=torch_gpu.bfloat16, device="cuda")
    q[..., 0] = 3.8125  # a logit of 15.25, e^-15.25 = 2^-22.0
    R.check(torch_gpu, p, q, q.double().cpu().numpy(), "bf16", scale=1.0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", [900, 960, 1000, 1023, 1024, 1087, 1100, 1152, 2048, 2899])
@pytest.mark.parametrize("most,kind", [(40, "splits"), (9000, "chunk"), (4, "shares")])
def test_a_value_past_fp16_around_a_window_of_pages(torch_gpu, d, at, most, kind):
    """The tokens' pages are looked up 64 at a time, ahead of the tile at work: the loop that goes on from a tile with
    such a value may have to go back to pages before them."""
    rng = np.random.default_rng(at)
    new = min(most, 40)
    p = Pool(torch_gpu, d, [0, new], [2900], 1, 16, 4, seed=at, max_new=most, extra_cols=60)
    assert plan(p.shape, d).kind == kind
    R.spread(p, rng)
    p.host["v_scales"][p.table[0, at // 16], 0, at % 16, 1] = 60
    p.upload()
    q, qv = R.queries(torch_gpu, rng, p, "bf16")
    R.check(torch_gpu, p, q, qv, "bf16")
