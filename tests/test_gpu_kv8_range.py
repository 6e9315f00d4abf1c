"""Attention on the 8-bit cache when one row takes most of the weight and its value is zero, as good as an
attention sink's: the output is then that of the other rows, however small their weights are.

The dominant score is exact by construction, so that only the weights' own rounding is seen: the rotary
tables are the identity and the rotary query is +-1, alike in all heads, so the row's rotary part sets the same
score for every head without a rounding. Bounds: the element bound of check_out, whose `mag` the rows behind
fill here, and the relative 2-norm of 2^-8 that the steps of the other tests are held to (independent
errors of up to 2^-8 per probability and 2^-9 of the output's own rounding)."""
import numpy as np
import pytest
import torch

import kv8_testlib as R
from mla_testlib import fleet
from test_gpu_kv8 import CFG, Step, make_cache, random_rows

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def sink_step(dev, n, seed, nats, at=0, mate=None, **kw):
    """A step over n rows N(0, 1); row `at` has a latent part of zeros and a score of `nats` for every
    head. mate = f: the row after it is f times larger and has a score of -20 nats."""
    st = Step(dev, [n], seed, **kw)
    st.cos = st.runner.cos = torch.ones_like(st.cos)
    st.sin = st.runner.sin = torch.zeros_like(st.sin)
    q = st.q.view(1, 16, 192)
    sign = torch.where(torch.arange(64, device=dev) * 37 % 64 < 32, 1.0, -1.0).to(BF)
    q[:, :, 128:] = sign
    k = torch.cat([sign[0::2], sign[1::2]]).float().cpu() / (64 * CFG.softmax_scale)  # a score of one nat
    x = random_rows(n, seed + 1).float()
    x[at, :512] = 0
    x[at, 512:] = k * nats
    if mate is not None:
        x[at + 1, :512] *= mate
        x[at + 1, 512:] = -20 * k
    rows = x.to(BF)
    cache = make_cache([n], dev, seed + 2)
    fleet.rows_to_pages(cache, rows.to(dev), [0, n], [0])
    want = R.Cache8(n + 1)
    want.write(0, rows.double().numpy())
    out = st.runner.attend(st.q, st.kv_a, cache, check="sync")
    want.write(n, st.new_row(0))
    st.check(out, lambda b: want.values(n + 1), f"{n} rows, {nats} nats")
    return st, cache, out


@pytest.mark.parametrize("ctas", [1, 0])
@pytest.mark.parametrize("n,nats", [(200, 12), (4096, 10.6), (4096, 14), (16384, 11.9), (16384, 12.8), (60000, 12.5),
                                    (60000, 16)])
def test_rows_behind_a_dominant_one(cuda_device, n, nats, ctas):
    """The others have 2^-15 to 2^-23 of the dominant weight each."""
    sink_step(cuda_device, n, 700, nats, num_ctas=ctas)


@pytest.mark.parametrize("at", [40, 2000, 4095])
def test_a_dominant_row_anywhere(cuda_device, at):
    """The rows before it were weighted under a smaller reference."""
    sink_step(cuda_device, 4096, 710, 13, at=at, num_ctas=1)


@pytest.mark.parametrize("mate", [16.0, 64.0])
def test_a_dominant_row_beside_a_large_one(cuda_device, mate):
    """A block whose scale is set by a row without weight: the dominant probability is held larger by that scale."""
    sink_step(cuda_device, 4096, 720, 13, mate=mate, num_ctas=1)


def test_a_sink_before_a_window(cuda_device):
    sink_step(cuda_device, 9000, 730, 13, window=4096, sinks=4, num_ctas=1)
    sink_step(cuda_device, 9000, 730, 13, window=4096, sinks=4)
