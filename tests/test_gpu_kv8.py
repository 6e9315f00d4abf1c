"""The 8-bit latent cache on the GPU: rows stored and read back, the decode step's append and
its attention, against 64-bit restatements (kv8_testlib)."""
import importlib

import numpy as np
import pytest
import torch

import kv8_testlib as R
from mla_testlib import fleet, workloads

pytestmark = pytest.mark.gpu
native = importlib.import_module("fleet-mi300x_b200.native")
BF = torch.bfloat16
CFG = fleet.ModelConfig()


def make_cache(lens, dev, seed, garbage=True, extra=1):
    """An 8-bit cache with pages in random order; every byte and exponent that no row fills is a
    NaN or an extreme."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(n + extra) // 64) for n in lens]
    total = sum(need) + 2
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need)), -7, dtype=torch.int32)
    off = 0
    for b, n in enumerate(need):
        table[b, :n] = order[off:off + n]
        off += n
    cache = fleet.PagedLatentCache8(total, len(lens), max(need), device=dev)
    cache.block_table.copy_(table)
    cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    if garbage:
        cache.pages.fill_(0x7F)
        cache.pages[:, ::3] = 0xFF
        cache.scales.fill_(-128)
        cache.scales[::2] = 127
    return cache


def random_rows(n, seed, spread=0.0):
    """bf16 rows N(0, 1), each scaled by 2^U(-spread, spread)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, 576, generator=g)
    return (x * torch.exp2((torch.rand(n, 1, generator=g) * 2 - 1) * spread)).to(BF)


def fill(cache, lens, seed, spread=0.0):
    """Rows 0 .. lens[b] - 1 of every request, in one call; their 64-bit restatements."""
    rows = random_rows(max(1, sum(lens)), seed, spread)
    starts = np.concatenate([[0], np.cumsum(lens)])
    fleet.rows_to_pages(cache, rows.to(cache.device), starts, [0] * len(lens))
    want = []
    for b, n in enumerate(lens):
        c = R.Cache8(n + 40)
        c.write(0, rows[starts[b]:starts[b + 1]].double().numpy())
        want.append(c)
    return want


# ------------------------------------------------------------------------------- rows
@pytest.mark.parametrize("lens,first", [
    ([1], [0]), ([16], [0]), ([17], [0]), ([64], [0]), ([200], [0]),
    ([0, 5, 0, 33, 1, 0], [3, 0, 7, 15, 16, 0]), ([1] * 40, list(range(40))), ([130, 2, 70], [61, 63, 1])])
def test_rows_are_stored_exactly(cuda_device, lens, first):
    """Bytes and exponents equal the definition's, the second call joining the first one's blocks."""
    cache = make_cache([a + b for a, b in zip(lens, first)], cuda_device, 1)
    before = fill(cache, first, 2, spread=2)
    rows = random_rows(max(1, sum(lens)), 3, spread=3)
    starts = np.concatenate([[0], np.cumsum(lens)])
    fleet.rows_to_pages(cache, rows.to(cuda_device), starts, first)
    for b, (n, f) in enumerate(zip(lens, first)):
        want = before[b]
        want.codes = np.concatenate([want.codes, np.zeros((n + 32, 576))])
        want.exps = np.concatenate([want.exps, np.zeros((n // 16 + 2, 2), np.int64)])
        want.write(f, rows[starts[b]:starts[b + 1]].double().numpy())
        codes, exps = R.read_request(cache, b, f + n)
        assert np.array_equal(exps, want.exps[:len(exps)]), b
        assert np.array_equal(codes, want.codes[:f + n]), b


def test_rows_of_every_magnitude(cuda_device):
    """Blocks of zeros, of the smallest and largest bf16 magnitudes, amax on both sides of a scale's
    limit, infinities and NaN."""
    rows = torch.zeros(16 * 8, 576)
    rows[16:32, 5] = 448.0
    rows[32:48, 5] = 450.0                       # one bf16 step above 448
    rows[48:64] = torch.randn(16, 576) * 1e-38
    rows[64:80] = torch.randn(16, 576) * 3e37
    rows[80:96] = torch.randn(16, 576)
    rows[85, 3], rows[86, 4], rows[87, 5], rows[88, 570] = float("inf"), -float("inf"), float("nan"), float("inf")
    rows[96:112] = torch.exp2(torch.linspace(-30, 8, 576))[None]
    rows[112:128] = torch.finfo(BF).max
    rows = rows.to(BF)
    cache = make_cache([128], cuda_device, 4)
    fleet.rows_to_pages(cache, rows.to(cuda_device), [0, 128], [0])
    want = R.Cache8(128)
    want.write(0, rows.double().numpy())
    codes, exps = R.read_request(cache, 0, 128)
    assert np.array_equal(exps, want.exps)
    assert np.array_equal(codes, want.codes, equal_nan=True)
    assert exps[0].tolist() == [-64, -64] and exps[1, 0] == 0 and exps[2, 0] == 1
    assert np.isnan(codes).sum() == 4


@pytest.mark.parametrize("stride", [576, 640, 3648])
def test_raw_rows_and_strides(cuda_device, stride):
    """RAW rows are the bf16 cache's rows, then rounded; rows may be a view of wider ones."""
    lens, first = [70, 0, 9], [5, 3, 60]
    lw = workloads.make_layer_weights(7, norm="uniform")
    cos, sin = fleet.device_rope_tables(CFG, 256, cuda_device)
    wide = torch.randn(79, stride, generator=torch.Generator().manual_seed(5)).to(BF).to(cuda_device)
    rows = wide[:, stride - 576:]
    starts = [0, 70, 70, 79]
    kw = dict(raw=True, norm_w=lw.kv_a_layernorm.to(cuda_device), cos=cos, sin=sin)
    cache = make_cache([a + b for a, b in zip(lens, first)], cuda_device, 6)
    ref = fleet.PagedLatentCache(cache.n_pages, 3, cache.max_blocks, device=cuda_device)
    ref.block_table.copy_(cache.block_table)
    fleet.rows_to_pages(ref, rows, starts, first, **kw)
    fleet.rows_to_pages(cache, rows, torch.tensor(starts, device=cuda_device), first, total=79, **kw)
    for b in (0, 2):
        want = R.Cache8(first[b] + lens[b])
        want.exps[:] = R.read_request(cache, b, first[b] + lens[b])[1] if first[b] % 16 else 0
        new = ref.read_rows(b, first[b], lens[b]).double().cpu().numpy()
        codes, exps = R.read_request(cache, b, first[b] + lens[b])
        for p in range(first[b] // 16 + 1, len(exps)):  # blocks that hold new rows only
            blk = new[max(0, p * 16 - first[b]):(p + 1) * 16 - first[b]]
            for k, (lo, hi) in enumerate(R.PARTS):
                e = R.exponent(blk[:, lo:hi])
                assert exps[p, k] == e
                assert np.array_equal(codes[p * 16:p * 16 + len(blk), lo:hi], R.round_e4m3(blk[:, lo:hi] * 2.0 ** -e))


def test_rows_reports_bad_positions_and_pages(cuda_device):
    cache = make_cache([70, 10], cuda_device, 8)
    word = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    rows = random_rows(40, 9).to(cuda_device)
    before = cache.pages.clone()
    fleet.rows_to_pages(cache, rows[:16], [0, 0, 16], [0, 120], error_word=word)  # past the block table
    assert int(word) == 2
    word.zero_()
    fleet.rows_to_pages(cache, rows[:4], [0, 0, 4], [0, -20], error_word=word)
    assert int(word) == 2
    word.zero_()
    cache.block_table[1, 0] = cache.n_pages
    fleet.rows_to_pages(cache, rows[:4], [0, 0, 4], [0, 0], error_word=word)
    assert int(word) == 1
    assert torch.equal(cache.pages, before)


# ------------------------------------------------------------------------------- the step
class Step:
    """A runner, inputs and the 64-bit restatement of one decode step."""

    def __init__(self, dev, lens, seed, window=0, sinks=0, num_ctas=0, max_pos=None, scale_q=1.0):
        self.lens, self.window, self.sinks = lens, window, sinks
        B = len(lens)
        lw = workloads.make_layer_weights(seed, norm="uniform")
        self.cos, self.sin = fleet.device_rope_tables(CFG, max_pos or max(lens) + 40, dev)
        w = fleet.LayerWeights(*(t.to(dev) for t in (lw.q_proj, lw.kv_a_proj_with_mqa, lw.kv_a_layernorm, lw.kv_b_proj,
                                                     lw.o_proj)))
        self.runner = fleet.MlaDecodeAttention(CFG, w, self.cos, self.sin, num_ctas=num_ctas, window=window, sinks=sinks)
        g = torch.Generator().manual_seed(seed + 1)
        self.q = (torch.randn(B, 3072, generator=g) * scale_q).to(BF).to(dev)
        self.kv_a = torch.randn(B, 576, generator=g).to(BF).to(dev)
        self.kv_b = lw.kv_b_proj.double().numpy()
        self.norm = lw.kv_a_layernorm.double().numpy()

    def new_row(self, b):
        """Request b's appended bf16 row, taken from a bf16 cache's step (its arithmetic has its own tests)."""
        one = fleet.PagedLatentCache(1, 1, 1, device=self.q.device)
        n = self.lens[b]
        runner = fleet.MlaDecodeAttention(CFG, self.runner.w, self.cos[n:n + 1], self.sin[n:n + 1])
        runner.attend(self.q[b:b + 1], self.kv_a[b:b + 1], one)
        return one.read_rows(0, 0, 1).double().cpu().numpy()

    def check(self, out, rows_of, what=""):
        out = out.double().cpu().numpy()
        cos, sin = self.cos.double().cpu().numpy(), self.sin.double().cpu().numpy()
        q = self.q.double().cpu().numpy()
        off = norm = 0.0
        for b, n in enumerate(self.lens):
            seen = R.visible(n, self.window, self.sinks)
            want, mag, ds = R.attention(q[b], rows_of(b)[seen], self.kv_b, cos[n], sin[n], CFG.softmax_scale)
            R.check_out(out[b], want, mag, ds, f"{what} request {b} of {n} rows")
            off += ((out[b] - want) ** 2).sum()
            norm += (want ** 2).sum()
        assert off <= (2.0 ** -8) ** 2 * norm, f"{what}: relative 2-norm {np.sqrt(off / norm):.2e}"


def run8(dev, lens, seed, spread=0.0, **kw):
    st = Step(dev, lens, seed, **kw)
    cache = make_cache(lens, dev, seed + 2)
    want = fill(cache, lens, seed + 3, spread)
    out = st.runner.attend(st.q, st.kv_a, cache, check="sync")
    for b, n in enumerate(lens):
        want[b].write(n, st.new_row(b))
        codes, exps = R.read_request(cache, b, n + 1)
        assert np.array_equal(exps, want[b].exps[:len(exps)]), f"request {b}: exponents after the append"
        assert np.array_equal(codes, want[b].codes[:n + 1]), f"request {b}: rows after the append"
    st.check(out, lambda b: want[b].values(lens[b] + 1))
    return st, cache, out


@pytest.mark.parametrize("lens", [
    [0], [1], [15], [16], [31], [62], [63], [64], [65], [126], [127], [128], [129], [1000],
    [0, 1, 63, 64, 127, 128, 300, 5], list(range(0, 140, 2))])
def test_step_matches_64_bits(cuda_device, lens):
    """Lengths around every boundary of a row block, page and tile; more than 64 requests too."""
    run8(cuda_device, lens, 20)


@pytest.mark.parametrize("ctas", [1, 2, 7, 148, 300])
def test_step_on_any_split(cuda_device, ctas):
    run8(cuda_device, [700, 3, 64, 1500, 129], 30, num_ctas=ctas)


def test_step_over_long_rows(cuda_device):
    run8(cuda_device, [20000], 40)


def test_rows_of_unlike_magnitude(cuda_device):
    """Rows 2^-6 .. 2^6 times the usual: blocks' scales differ, scores grow past the running reference."""
    run8(cuda_device, [900, 77, 300], 50, spread=6.0)


def test_sharp_scores(cuda_device):
    """Large queries: one row takes nearly all the weight, and the running maximum moves often. The
    error of a bf16 query grows with the scores, so only the element bound applies."""
    st = Step(cuda_device, [600, 90], 60, scale_q=4.0)
    cache = make_cache(st.lens, cuda_device, 61)
    want = fill(cache, st.lens, 62)
    out = st.runner.attend(st.q, st.kv_a, cache, check="sync").double().cpu().numpy()
    cos, sin = st.cos.double().cpu().numpy(), st.sin.double().cpu().numpy()
    for b, n in enumerate(st.lens):
        want[b].write(n, st.new_row(b))
        R.check_out(out[b], *R.attention(st.q[b].double().cpu().numpy(), want[b].values(n + 1), st.kv_b, cos[n], sin[n],
                                         CFG.softmax_scale))


def test_increasing_scores(cuda_device):
    """Rows whose score rises along the sequence: the reference is raised in every tile."""
    n = 1200
    st = Step(cuda_device, [n], 63)
    cache = make_cache([n], cuda_device, 64)
    q = st.q[0].double().cpu().numpy().reshape(16, 192)
    w = st.kv_b.reshape(16, 256, 512)
    qa = np.einsum("hd,hdc->hc", q[:, :128], w[:, :128])
    d = qa[3] / np.abs(qa[3]).max()
    x = np.random.RandomState(0).randn(n, 576)
    x[:, :512] += d[None] * np.linspace(0, 12, n)[:, None]
    rows = torch.from_numpy(x).to(BF)
    fleet.rows_to_pages(cache, rows.to(cuda_device), [0, n], [0])
    out = st.runner.attend(st.q, st.kv_a, cache, check="sync").double().cpu().numpy()
    want = R.Cache8(n + 1)
    want.write(0, rows.double().numpy())
    want.write(n, st.new_row(0))
    R.check_out(out[0], *R.attention(st.q[0].double().cpu().numpy(), want.values(n + 1), st.kv_b,
                                     st.cos[n].double().cpu().numpy(), st.sin[n].double().cpu().numpy(), CFG.softmax_scale))


def test_decode_loop_grows_scales(cuda_device):
    """40 steps whose rows grow: blocks are held anew under larger scales, as the definition does."""
    lens = [0, 9, 60]
    st = Step(cuda_device, lens, 70)
    cache = make_cache(lens, cuda_device, 71, extra=41)
    want = fill(cache, lens, 72)
    for step in range(40):
        st.kv_a = (torch.randn(3, 576, generator=torch.Generator().manual_seed(step)) * 1.3 ** step).to(BF).to(cuda_device)
        st.lens = [n + step for n in lens]
        out = st.runner.attend(st.q, st.kv_a, cache, check="sync")
        for b in range(3):
            want[b].codes = np.concatenate([want[b].codes, np.zeros((16, 576))])
            want[b].exps = np.concatenate([want[b].exps, np.zeros((1, 2), np.int64)])
            want[b].write(st.lens[b], st.new_row(b))
        cache.advance()
    for b in range(3):
        codes, exps = R.read_request(cache, b, lens[b] + 40)
        assert np.array_equal(exps, want[b].exps[:len(exps)])
        assert np.array_equal(codes, want[b].codes[:lens[b] + 40])
    st.check(out, lambda b: want[b].values(st.lens[b] + 1))


def test_outputs_repeat_bit_for_bit(cuda_device):
    st, cache, out = run8(cuda_device, [2000, 64, 513, 7], 80)
    for _ in range(5):
        assert torch.equal(st.runner.attend(st.q, st.kv_a, cache, check="sync"), out)


def test_streams_views_and_graphs(cuda_device):
    """Strided q / kv_a / out, another stream, a captured graph: the bits of the plain call."""
    st, cache, out = run8(cuda_device, [300, 65], 90)
    both = torch.zeros(2, 4000, dtype=BF, device=cuda_device)
    both[:, 100:3172], both[:, 3200:3776] = st.q, st.kv_a
    wide = torch.zeros(2, 2100, dtype=BF, device=cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        st.runner.attend(both[:, 100:3172], both[:, 3200:3776], cache, wide[:, 20:2068], check="sync")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(wide[:, 20:2068], out) and not wide[:, :20].any() and not wide[:, 2068:].any()
    graph = fleet.DecodeGraph(st.runner, cache, inputs="qkv", q=st.q, kv_a=st.kv_a)
    assert torch.equal(graph.replay(), out)


def test_attention_block_on_an_8_bit_cache(cuda_device):
    """K0 through K5 on the 8-bit cache equals its parts, the projections taken from a bf16 step."""
    lens = [100, 7]
    st = Step(cuda_device, lens, 95)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 2048, generator=g).to(BF).to(cuda_device)
    h = torch.randn(2, 2048, generator=g).to(BF).to(cuda_device)
    a, b = (make_cache(lens, cuda_device, 96) for _ in range(2))
    fill(a, lens, 97)
    fill(b, lens, 97)
    out = torch.empty(2, 2048, dtype=BF, device=cuda_device)
    st.runner.attention_block(x, a, h, out=out, check="sync")
    assert torch.equal(st.runner.attend_x(x, b, check="sync"), out)
    assert torch.equal(a.pages, b.pages) and torch.equal(a.scales, b.scales)


def test_sharded_step_on_an_8_bit_cache(cuda_device):
    """A sequence split in two shards (no new row in the first), combined: the whole's 64-bit value."""
    n, cut = 500, 192
    st = Step(cuda_device, [n], 100)
    rows = random_rows(n, 101)
    want = R.Cache8(n + 1)
    want.write(0, rows.double().numpy())
    want.write(n, st.new_row(0))
    parts = []
    for lo, hi in ((0, cut), (cut, n)):
        cache = make_cache([hi - lo], cuda_device, 102)
        fleet.rows_to_pages(cache, rows[lo:hi].to(cuda_device), [0, hi - lo], [0])
        part = torch.empty(1, 16, native.SHARD_STRIDE, device=cuda_device)
        st.runner.attend(st.q, st.kv_a, cache, rope_pos=torch.tensor([n], dtype=torch.int32, device=cuda_device),
                         shard_out=part, new_row=hi == n, check="sync")
        parts.append(part)
    st.check(fleet.combine_shards(torch.stack(parts)), lambda b: want.values(n + 1))


def test_non_finite_queries_stay_in_their_head(cuda_device):
    st, cache, out = run8(cuda_device, [200], 110)
    q = st.q.clone()
    q[0, 5 * 192 + 130] = float("nan")
    q[0, 9 * 192 + 150] = float("inf")
    got = st.runner.attend(q, st.kv_a, cache, check="sync").view(16, 128)
    finite = torch.isfinite(got).all(1).tolist()
    assert finite == [h not in (5, 9) for h in range(16)]


def test_device_errors(cuda_device):
    """A bad page and a bad position are reported; requests beside them keep their outputs."""
    st, cache, out = run8(cuda_device, [200, 90, 40], 120)
    cache.seq_lens[1] = -3
    got = torch.zeros_like(out)
    st.runner.attend(st.q, st.kv_a, cache, got, check=False)
    with pytest.raises(native.MlaError):
        st.runner.check_errors()
    assert torch.equal(got[0], out[0]) and torch.equal(got[2], out[2])
    cache.seq_lens[1] = 90
    keep = cache.block_table[1, 0].clone()
    cache.block_table[1, 0] = cache.n_pages + 5
    st.runner.attend(st.q, st.kv_a, cache, got, check=False)
    with pytest.raises(native.MlaError):
        st.runner.check_errors()
    cache.block_table[1, 0] = keep
    assert torch.equal(st.runner.attend(st.q, st.kv_a, cache, check="sync"), out)


def test_refusals(cuda_device):
    dev = cuda_device
    st, cache, _ = run8(dev, [30], 130)
    for kw in (dict(check_kernel=True), dict(kernel="tcgen05"), dict(qc_hilo=True), dict(p_hilo=True)):
        r = fleet.MlaDecodeAttention(CFG, st.runner.w, st.cos, st.sin, **kw)
        with pytest.raises(native.MlaError):
            r.attend(st.q, st.kv_a, cache)
    p = st.runner.params(st.q, st.kv_a, cache, torch.empty(1, 2048, dtype=BF, device=dev))
    for field, value, code in (("kv_scales", None, -1), ("kv_scales", cache.scales.data_ptr() + 4, -3),
                               ("uk_norm", None, -1), ("window", -1, -1), ("sinks", 3, -1)):
        keep = getattr(p, field)
        setattr(p, field, value)
        assert st.runner.lib.mla_decode_step(p, None) == code, field
        setattr(p, field, keep)
    p.flags &= ~native.FLAG_KV8
    assert st.runner.lib.mla_decode_step(p, None) == -1  # exponents without the flag
    with pytest.raises(ValueError):
        fleet.rows_to_pages(cache, torch.zeros(4, 576, device=dev), [0, 4])  # not bf16
    with pytest.raises(ValueError):
        fleet.rows_to_pages(cache, torch.zeros(4, 576, dtype=BF), [0, 4])  # rows on the host
    with pytest.raises(ValueError):
        fleet.rows_to_pages(cache, torch.zeros(4, 576, dtype=BF, device=dev), [0, 5])
    with pytest.raises(native.MlaError):
        fleet.rows_to_pages(cache, torch.zeros(4, 576, dtype=BF, device=dev), [0, 4], total=-1)
    with pytest.raises(ValueError):
        fleet.PagedLatentCache8.from_tensors(cache.pages[:, :100], cache.scales, cache.block_table, cache.seq_lens)


def test_static_step(cuda_device):
    """The step with the library's own workspace: the bits of the step with the caller's."""
    st, cache, out = run8(cuda_device, [200, 9], 150)
    got = torch.empty_like(out)
    p = st.runner.params(st.q, st.kv_a, cache, got)
    native.check(st.runner.lib.mla_decode_step_static(p, torch.cuda.current_stream().cuda_stream), "static", p)
    torch.cuda.synchronize()
    assert torch.equal(got, out)


def test_uk_norms(cuda_device):
    """The largest column norm of every head's W_UK: fp32 sums of 128 squares, then a root, 2^-16 relative at most."""
    w = workloads.make_layer_weights(9).kv_b_proj
    got = torch.empty(16, device=cuda_device)
    lib = native.load_library()
    kv_b = w.to(cuda_device)
    assert lib.mla_uk_norms(kv_b.data_ptr(), got.data_ptr(), None) == 0
    torch.cuda.synchronize()
    want = w.double().view(16, 256, 512)[:, :128].norm(dim=1).amax(1)
    assert ((got.cpu().double() - want).abs() <= want * 2.0 ** -16).all()
    assert lib.mla_uk_norms(None, got.data_ptr(), None) == -1
    assert lib.mla_uk_norms(kv_b.data_ptr() + 2, got.data_ptr(), None) == -3


def test_zero_and_tiny_queries(cuda_device):
    """A query of zeros attends evenly; one far below bf16's usual range keeps its values (the bounds follow
    from the derivation in check_out: they scale with the scores)."""
    st, cache, _ = run8(cuda_device, [100, 70], 160)
    codes = [R.read_request(cache, b, n + 1) for b, n in enumerate(st.lens)]
    values = []
    for c, e in codes:
        f = np.exp2(np.repeat(e.astype(np.float64), 16, 0))[:len(c)]
        values.append(c * np.concatenate([np.repeat(f[:, :1], 512, 1), np.repeat(f[:, 1:], 64, 1)], 1))
    for scale in (0.0, 1e-12):
        st.q = (st.q.float() * scale).to(BF)
        out = st.runner.attend(st.q, st.kv_a, cache, check="sync")
        st.check(out, lambda b: values[b], f"scale {scale}")
        st.q = torch.randn(2, 3072, generator=torch.Generator().manual_seed(161)).to(BF).to(cuda_device)


def test_read_and_write_rows_helpers(cuda_device):
    cache = make_cache([100, 20], cuda_device, 140)
    rows = random_rows(37, 141)
    cache.write_rows(1, 0, rows[:20])
    cache.write_rows(0, 0, rows)
    want = R.Cache8(37)
    want.write(0, rows.double().numpy())
    got = cache.read_rows(0, 0, 37)
    assert got.dtype == torch.float32 and np.array_equal(got.double().cpu().numpy(), want.values(37))


@pytest.mark.parametrize("kind", ["decode", "stack"])
def test_setting_up_a_graph_leaves_the_rows_alone(cuda_device, kind):
    """The set-up's step stores a row of whatever the buffers hold; a large one must not coarsen the started
    block's earlier rows for good. The first replay equals the eager step on an untouched cache."""
    lens = [37, 64, 5]
    st = Step(cuda_device, lens, 170)
    a, b = (make_cache(lens, cuda_device, 171) for _ in range(2))
    for cache in (a, b):
        fill(cache, lens, 172)
    before = a.pages.clone(), a.scales.clone()
    want = st.runner.attend(st.q, st.kv_a, b, check="sync").clone()
    q, kv = torch.randn_like(st.q), torch.randn_like(st.kv_a) * 1e6
    if kind == "decode":
        graph = fleet.DecodeGraph(st.runner, a, inputs="qkv", q=q, kv_a=kv)
    else:
        graph = fleet.LayerStackGraph([st.runner], [a], mode="slice", q=[q], kv_a=[kv])
    assert torch.equal(a.pages, before[0]) and torch.equal(a.scales, before[1])
    q.copy_(st.q)
    kv.copy_(st.kv_a)
    out = graph.replay()
    graph.synchronize()
    assert torch.equal(out if kind == "decode" else graph.out[0], want)
    for r, n in enumerate(lens):
        assert np.array_equal(R.read_request(a, r, n + 1)[1], R.read_request(b, r, n + 1)[1])
        assert np.array_equal(R.read_request(a, r, n + 1)[0], R.read_request(b, r, n + 1)[0])


def test_write_rows_reports_rows_it_cannot_store(cuda_device):
    cache = make_cache([70, 10], cuda_device, 180)
    before = cache.pages.clone()
    with pytest.raises(native.MlaError) as e:
        cache.write_rows(1, 130, random_rows(20, 181))  # past the block table
    assert e.value.code == 2
    cache.block_table[0, 1] = cache.n_pages
    with pytest.raises(native.MlaError) as e:
        cache.write_rows(0, 64, random_rows(5, 182))
    assert e.value.code == 1
    assert torch.equal(cache.pages, before)


@pytest.mark.parametrize("bits,batch", [(8, 3), (16, 3), (16, 70)])
def test_counts_changed_right_before_a_step(cuda_device, bits, batch):
    """Row counts written by the kernel in front of the step (advance), many steps without a wait: every row at its
    position, outputs as with a wait between."""
    steps = 200
    st = Step(cuda_device, [0] * batch, 190, max_pos=steps + 8)
    cls = fleet.PagedLatentCache8 if bits == 8 else fleet.PagedLatentCache
    a, b = (cls.for_lengths([0] * batch, extra_tokens=steps, permute=False, device=cuda_device) for _ in range(2))
    g = torch.Generator().manual_seed(191)
    kv = torch.randn(steps, batch, 576, generator=g).to(BF).to(cuda_device)
    got, want = (torch.empty(steps, batch, 2048, dtype=BF, device=cuda_device) for _ in range(2))
    for k in range(steps):
        st.runner.attend(st.q, kv[k], a, got[k])
        a.advance()
    for k in range(steps):
        st.runner.attend(st.q, kv[k], b, want[k], check="sync")
        b.advance()
        torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(a.pages, b.pages)
