"""The softmax weights of the attention over picked pages in its second product, in steps and in chunks of rows alike:
two bf16 parts of each, whatever the output's type."""
from __future__ import annotations

import numpy as np
import pytest

from cache_rows import tolerance
from test_gpu_cache import Pool
from test_gpu_pick import attend, plan, run_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("most", [60, 1100])
@pytest.mark.parametrize("q_type,out_type", [("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f16")])
def test_values_that_nearly_cancel(torch_gpu, d, page, most, q_type, out_type):
    """Every second token has the logit 0 and values of 1, the others -x and values of -1: the output is about x / 2, and
    the rounding of the weight e^-x, which an output of that size does not hide, is all that it can be off by. Keys are zero
    but in one channel, so that a logit is one exact product: tolerance's terms for logits are nothing here. Weights
    of 11 bits have steps of 2^-11 below 1 and move an output by up to 2^-13: past the bound."""
    torch = torch_gpu
    rng = np.random.default_rng(page + d)
    p = Pool(torch, d, [0, 60, 61], [128, 64], 2, page, 8, extra_cols=1, seed=page, max_new=most)
    top = p.table.shape[1]
    assert plan(p.shape, d, top).chunks == (most == 1100)
    for side in "kv":
        p.host[side + "_codes"][:] = 0
        p.host[side + "_scales"][:] = 127
    p.host["k_codes"][:, :, 1::2, 0] = 0x0a  # -1.0 in channel 0
    p.host["v_codes"][:, :, ::2] = 0x22      # 1.0
    p.host["v_codes"][:, :, 1::2] = 0xaa     # -1.0
    p.upload()
    q = torch.zeros(1, p.rows, 8, d, device="cuda")
    q[..., 0] = torch.from_numpy(2.0 ** -8 * (1 + rng.random((p.rows, 8)))).cuda()
    q = q.to(torch.bfloat16 if q_type == "bf16" else torch.float16)
    picked = np.broadcast_to(np.arange(top), (p.rows, 2, top)).astype(np.int32).copy()
    picked[::3, :, 0] = -1  # rows that have not picked the first page, in units with rows that have
    got = run_attend(torch, p, q, picked, out_type, causal=False, scale=1.0)[0].double().cpu().numpy()
    want, size, reach, count, most_v = attend(p, q[0].double().cpu().numpy(), picked, False, 1.0, np.full(got.shape, 3.0))
    tol = tolerance(want, size, reach, count, most_v, d, out_type, False)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), bad.size, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])
