"""A runner whose kv_b changes, on the 8-bit cache: the scale of the query follows the weights, however they
were replaced and wherever the step runs."""
import pytest
import torch

from mla_testlib import fleet
from test_gpu_kv8 import CFG, Step, fill, make_cache

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
LENS = [300, 70]


def fresh(st, cache_seed, dev):
    """What a runner made with the current weights computes."""
    runner = fleet.MlaDecodeAttention(CFG, st.runner.w, st.cos, st.sin)
    cache = make_cache(LENS, dev, cache_seed)
    fill(cache, LENS, cache_seed + 1)
    return runner.attend(st.q, st.kv_a, cache, check="sync")


def start(dev, seed):
    st = Step(dev, LENS, seed)
    cache = make_cache(LENS, dev, seed + 2)
    fill(cache, LENS, seed + 3)
    first = st.runner.attend(st.q, st.kv_a, cache, check="sync").clone()
    return st, cache, first


@pytest.mark.parametrize("factor", [8.0, 2.0 ** -12])
def test_weights_updated_in_place(cuda_device, factor):
    """Larger columns would saturate the query's pairs under the old scale, smaller ones lose their bits."""
    st, cache, first = start(cuda_device, 800)
    st.runner.kv_b[:].mul_(factor)  # a power of two, and a view: the bits of a fresh runner
    got = st.runner.attend(st.q, st.kv_a, cache, check="sync")
    assert not torch.equal(got, first)
    assert torch.equal(got, fresh(st, 802, cuda_device))
    st.runner.kv_b.mul_(1 / factor)
    assert torch.equal(st.runner.attend(st.q, st.kv_a, cache, check="sync"), first)


def test_weights_replaced(cuda_device):
    st, cache, first = start(cuda_device, 810)
    st.runner.w.kv_b_proj = st.runner.kv_b = st.runner.kv_b * 8
    assert torch.equal(st.runner.attend(st.q, st.kv_a, cache, check="sync"), fresh(st, 812, cuda_device))


def test_weights_updated_between_replays(cuda_device):
    """A captured step reads the weights when it runs; so does the query's scale."""
    st, cache, first = start(cuda_device, 820)
    one = fleet.DecodeGraph(st.runner, cache, inputs="qkv", q=st.q, kv_a=st.kv_a)
    stack = fleet.LayerStackGraph([st.runner], [cache], mode="slice", q=[st.q], kv_a=[st.kv_a])
    assert torch.equal(one.replay(), first)
    st.runner.kv_b.mul_(8)
    want = fresh(st, 822, cuda_device)
    assert torch.equal(one.replay(), want)
    stack.replay()
    stack.synchronize()
    assert torch.equal(stack.out[0], want)
    st.runner.kv_b.mul_(0.125)
    stack.replay()
    assert torch.equal(stack.out[0], first)


def test_updates_that_torch_does_not_count(cuda_device):
    """Through .data the version counter stands still: update_norms says so; a tensor made in inference mode
    has no counter, and its norms are taken at every step."""
    st, cache, first = start(cuda_device, 830)
    st.runner.kv_b.data.mul_(8)
    st.runner.update_norms()
    want = fresh(st, 832, cuda_device)
    assert torch.equal(st.runner.attend(st.q, st.kv_a, cache, check="sync"), want)
    with torch.inference_mode():
        st.runner.kv_b = st.runner.kv_b * 0.125
    assert torch.equal(st.runner.attend(st.q, st.kv_a, cache, check="sync"), first)
    graph = fleet.DecodeGraph(st.runner, cache, inputs="qkv", q=st.q, kv_a=st.kv_a)
    with torch.inference_mode():
        st.runner.kv_b.mul_(8)
    assert torch.equal(st.runner.attend(st.q, st.kv_a, cache, check="sync"), want)
    assert torch.equal(graph.replay(), want)


def test_first_step_inside_a_capture(cuda_device):
    """A runner whose first step on an 8-bit cache is captured by the caller: replays and later eager steps agree."""
    st, cache, first = start(cuda_device, 840)
    other = fleet.PagedLatentCache.for_lengths(LENS, device=cuda_device)
    runner = fleet.MlaDecodeAttention(CFG, st.runner.w, st.cos, st.sin)
    out = torch.empty_like(first)
    need = runner.params(st.q, st.kv_a, cache, out)  # the workspace, before the capture
    runner.attend(st.q, st.kv_a, other, check="sync")
    runner = fleet.MlaDecodeAttention(CFG, st.runner.w, st.cos, st.sin)
    runner._ws = torch.empty(need.workspace_bytes, dtype=torch.uint8, device=cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        runner.attend(st.q, st.kv_a, cache, out)
    assert torch.equal(runner.attend(st.q, st.kv_a, cache, check="sync"), first)  # before any replay
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)


def test_first_step_on_another_stream(cuda_device):
    """The norms are taken on the step's stream, not on the constructor's: nothing has to be waited for."""
    st, cache, first = start(cuda_device, 850)
    busy = torch.randn(4096, 4096, device=cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        busy = busy @ busy  # the constructor's stream is behind
        busy /= busy.norm()
    runner = fleet.MlaDecodeAttention(CFG, st.runner.w, st.cos, st.sin)
    with torch.cuda.stream(side):
        got = runner.attend(st.q, st.kv_a, cache, check="sync")
    torch.cuda.synchronize()
    assert torch.equal(got, first)
