"""Sliding windows with sinks on the GPU, on both caches, against 64-bit restatements."""
import numpy as np
import pytest
import torch

import kv8_testlib as R
from mla_testlib import fleet
from test_gpu_kv8 import CFG, Step, fill, make_cache, native, random_rows, run8

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

WINDOWS = [(1, 0), (1, 1), (16, 0), (31, 1), (32, 4), (33, 63), (64, 64), (65, 65), (100, 130), (128, 0), (1000, 5),
           (5000, 3)]
LENS = [0, 1, 31, 32, 63, 64, 65, 100, 127, 130, 200, 257, 1023]


@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_window_on_an_8_bit_cache(cuda_device, window, sinks):
    run8(cuda_device, LENS, 200, window=window, sinks=sinks)


def bf16_cache(lens, dev, seed, nan=True):
    cache = fleet.PagedLatentCache.for_lengths(lens, spare_pages=2, generator=torch.Generator().manual_seed(seed), device=dev)
    if nan:
        cache.pages.fill_(float("nan"))
        cache.pages[:, ::2] = float("inf")
    rows = []
    for b, n in enumerate(lens):
        x = random_rows(max(n, 1), seed + b)[:n]
        if n:
            cache.write_rows(b, 0, x)
        rows.append(x.double().numpy())
    return cache, rows


def run16(dev, lens, seed, window, sinks, **kw):
    st = Step(dev, lens, seed, window=window, sinks=sinks, **kw)
    cache, rows = bf16_cache(lens, dev, seed + 5)
    out = st.runner.attend(st.q, st.kv_a, cache, check="sync")
    rows = [np.concatenate([rows[b], st.new_row(b)]) for b in range(len(lens))]
    st.check(out, lambda b: rows[b])
    return st, cache, out


@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_window_on_a_bf16_cache(cuda_device, window, sinks):
    run16(cuda_device, LENS, 300, window, sinks)


def test_window_for_many_requests(cuda_device):
    lens = [(37 * b) % 500 for b in range(100)]
    run8(cuda_device, lens, 310, window=90, sinks=2)
    run16(cuda_device, lens, 310, 90, 2)


@pytest.mark.parametrize("ctas", [1, 5, 296])
def test_window_on_any_split(cuda_device, ctas):
    run8(cuda_device, [900, 300, 40], 320, window=333, sinks=70, num_ctas=ctas)
    run16(cuda_device, [900, 300, 40], 320, 333, 70, num_ctas=ctas)


@pytest.mark.parametrize("hilo", [dict(qc_hilo=True), dict(p_hilo=True), dict(qc_hilo=True, p_hilo=True)])
def test_window_with_the_hilo_forms(cuda_device, hilo):
    st, cache, out = run16(cuda_device, [700, 90], 330, 150, 20)
    r = fleet.MlaDecodeAttention(CFG, st.runner.w, st.cos, st.sin, window=150, sinks=20, **hilo)
    got = r.attend(st.q, st.kv_a, cache, check="sync")
    assert (got.float() - out.float()).norm() <= 2.0 ** -7 * out.float().norm()


def test_a_window_of_everything_is_no_window(cuda_device):
    """window > rows: the bits of the step without one, on both caches."""
    lens = [300, 64, 1]
    for make in (lambda: make_cache(lens, cuda_device, 340), lambda: bf16_cache(lens, cuda_device, 340)[0]):
        cache = make()
        if isinstance(cache, fleet.PagedLatentCache8):
            fill(cache, lens, 341)
        plain = Step(cuda_device, lens, 342)
        wide = fleet.MlaDecodeAttention(CFG, plain.runner.w, plain.cos, plain.sin, window=1000, sinks=9)
        a = plain.runner.attend(plain.q, plain.kv_a, cache, check="sync")
        b = wide.attend(plain.q, plain.kv_a, cache, check="sync")
        assert torch.equal(a, b)


def test_unseen_rows_and_pages_are_not_read(cuda_device):
    """NaN rows outside the window leave no trace, and block-table entries of unseen pages may be anything."""
    for bits in (8, 16):
        st, cache, out = (run8(cuda_device, [1000], 350, window=200, sinks=10) if bits == 8 else
                          run16(cuda_device, [1000], 350, 200, 10))
        t = torch.arange(10, 801, device=cuda_device)
        page, slot = cache.block_table[0].long()[t // 64], t % 64
        if bits == 16:
            cache.pages[page, slot] = float("nan")
        else:
            cache.pages[:, :64 * 512].unflatten(1, (64, 512))[page, slot] = 0x7F
            cache.pages[:, 64 * 512:].unflatten(1, (64, 64))[page, slot] = 0xFF
        cache.block_table[0, 1:12] = 1 << 30
        assert torch.equal(st.runner.attend(st.q, st.kv_a, cache, check="sync"), out)


def test_window_in_a_graph_and_a_loop(cuda_device):
    """A captured step with advancing positions sees the window move."""
    lens = [120]
    st = Step(cuda_device, lens, 360, window=50, sinks=4)
    cache = make_cache(lens, cuda_device, 361, extra=30)
    eager = make_cache(lens, cuda_device, 361, extra=30)
    fill(cache, lens, 362)
    fill(eager, lens, 362)
    graph = fleet.DecodeGraph(st.runner, cache, inputs="qkv", q=st.q, kv_a=st.kv_a, advance=True)
    for _ in range(20):
        want = st.runner.attend(st.q, st.kv_a, eager, check="sync")
        eager.advance()
        assert torch.equal(graph.replay(), want)


def test_window_refusals(cuda_device):
    st, cache, _ = run8(cuda_device, [30], 370)
    w = st.runner.w
    for kw in (dict(window=-1), dict(sinks=4), dict(window=5, sinks=-1), dict(window=8, check_kernel=True),
               dict(window=8, kernel="tcgen05")):
        with pytest.raises(ValueError):
            fleet.MlaDecodeAttention(CFG, w, st.cos, st.sin, **kw)
    r = fleet.MlaDecodeAttention(CFG, w, st.cos, st.sin, window=8)
    part = torch.empty(1, 16, native.SHARD_STRIDE, device=cuda_device)
    with pytest.raises(native.MlaError):
        r.attend(st.q, st.kv_a, cache, shard_out=part)
    with pytest.raises(native.MlaError):
        r.attend(st.q, st.kv_a, cache, new_row=False)


@pytest.mark.parametrize("window,sinks", [(150, 20), (1000, 1)])
def test_the_hilo_forms_sharpen_a_window_too(cuda_device, window, sinks):
    """qc_hilo and p_hilo together under a window, against the 64-bit value. What is left is the output's
    rounding to bf16, as large as that of the 64-bit value itself (its 2-norm over 6,144 elements, to 5 %), and errors of
    about 2^-16 in q_c, the probabilities and fp32 sums, held to 2^-12 in all. The default form has bf16's
    rounding of q_c and of the probabilities besides and lies above that bound."""
    lens = [700, 90, 1500]
    st, cache, out = run16(cuda_device, lens, 380, window, sinks)
    r = fleet.MlaDecodeAttention(CFG, st.runner.w, st.cos, st.sin, window=window, sinks=sinks, qc_hilo=True, p_hilo=True)
    got = r.attend(st.q, st.kv_a, cache, check="sync").double().cpu().numpy()
    out = out.double().cpu().numpy()
    cos, sin = st.cos.double().cpu().numpy(), st.sin.double().cpu().numpy()
    off, plain, rounding, norm = 0.0, 0.0, 0.0, 0.0
    for b, n in enumerate(lens):
        rows = np.concatenate([cache.read_rows(b, 0, n).double().cpu().numpy(), st.new_row(b)])
        want = R.attention(st.q[b].double().cpu().numpy(), rows[R.visible(n, window, sinks)], st.kv_b, cos[n], sin[n],
                           CFG.softmax_scale)[0]
        off += ((got[b] - want) ** 2).sum()
        plain += ((out[b] - want) ** 2).sum()
        rounding += ((R.bf16(want) - want) ** 2).sum()
        norm += (want ** 2).sum()
    bound = 1.05 * rounding ** 0.5 + 2.0 ** -12 * norm ** 0.5
    assert off ** 0.5 <= bound < plain ** 0.5, (np.sqrt(off / norm), bound / norm ** 0.5, np.sqrt(plain / norm))
