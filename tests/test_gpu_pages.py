"""Fork, release, reserve, compact and copy of cache pages on the GPU, against a model in Python,
and a decode loop that uses them together."""
import random

import numpy as np
import pytest
import torch

import kv8_testlib as R
from mla_testlib import fleet
from test_gpu_kv8 import CFG, Step, native, random_rows

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class Model:
    """The definition: tables, counts and page contents (a tag per page and row) in Python."""

    def __init__(self, batch, n_pages, max_blocks, rows):
        self.n_pages, self.max_blocks = n_pages, max_blocks
        self.lens = [0] * batch
        self.tables = [[] for _ in range(batch)]
        self.tags = np.arange(n_pages * 64).reshape(n_pages, 64)  # which start row a row's bytes are
        order = random.Random(5).sample(range(n_pages), n_pages)
        for b, r in enumerate(rows):
            self.lens[b] = r
            self.tables[b] = [order.pop() for _ in range(-(-r // 64))]

    def refs(self):
        n = [0] * self.n_pages
        for t in self.tables:
            for p in t:
                n[p] += 1
        return n

    def free(self):
        return [p for p, n in enumerate(self.refs()) if n == 0]

    def fork(self, src, dst):
        free, new = self.free(), []
        last = {b: i for i, b in enumerate(dst)}
        pairs = [(a, b) for i, (a, b) in enumerate(zip(src, dst)) if a != b and last[b] == i]
        if len([1 for a, b in pairs if self.lens[a] % 64]) > len(free):
            return False
        for a, b in pairs:
            full, part = divmod(self.lens[a], 64)
            t = self.tables[a][:full]
            if part:
                p = free.pop(0)
                self.tags[p, :part] = self.tags[self.tables[a][full], :part]
                t = t + [p]
            new.append((b, t, self.lens[a]))
        for b, t, n in new:
            self.tables[b], self.lens[b] = t, n
        return True

    def release(self, requests):
        for b in requests:
            self.tables[b], self.lens[b] = [], 0

    def reserve(self, tokens, requests):
        need = [(b, max(0, -(-(self.lens[b] + tokens) // 64) - len(self.tables[b]))) for b in dict.fromkeys(requests)]
        free = self.free()
        if sum(n for _, n in need) > len(free):
            return False
        for b, n in need:
            self.tables[b] = self.tables[b] + [free.pop(0) for _ in range(n)]
        return True

    def compact(self):
        refs = self.refs()
        live = sum(n > 0 for n in refs)
        to = [p for p in range(live) if not refs[p]]
        from_ = [p for p in range(live, self.n_pages) if refs[p]]
        move = dict(zip(from_, to))
        for a, b in move.items():
            self.tags[b] = self.tags[a]
        self.tables = [[move.get(p, p) for p in t] for t in self.tables]


class Twin:
    """A PagePool over real caches, and the model beside it."""

    def __init__(self, dev, bits, layers, batch, n_pages, max_blocks, rows):
        self.m = Model(batch, n_pages, max_blocks, rows)
        table = torch.zeros(batch, max_blocks, dtype=torch.int32, device=dev)
        lens = torch.tensor(self.m.lens, dtype=torch.int32, device=dev)
        for b, t in enumerate(self.m.tables):
            table[b, :len(t)] = torch.tensor(t, dtype=torch.int32)
        tags = torch.from_numpy(self.m.tags).to(dev)
        self.caches = []
        for layer in range(layers):
            x = (tags + 7 * layer) & 0xFFFF
            if bits == 16:
                pages = (x[:, :, None] * 977 + torch.arange(576, device=dev)).to(torch.int16).view(BF)
                self.caches.append(fleet.PagedLatentCache.from_tensors(pages.contiguous(), table, lens))
            else:
                pages = torch.cat([(x[:, :, None] * 31 + torch.arange(512, device=dev)).flatten(1),
                                   (x[:, :, None] * 57 + torch.arange(64, device=dev)).flatten(1)], 1).to(torch.uint8)
                scales = x[:, ::16].repeat_interleave(2, 1).to(torch.int8).view(n_pages, 4, 2).contiguous()
                self.caches.append(fleet.PagedLatentCache8.from_tensors(pages.contiguous(), scales, table, lens))
        self.bits, self.start = bits, [c.pages.clone() for c in self.caches]
        self.scales = [c.scales.clone() for c in self.caches] if bits == 8 else None
        self.pool = fleet.PagePool(self.caches)

    def check(self):
        c = self.caches[0]
        assert c.seq_lens.tolist() == self.m.lens
        assert self.pool.held.tolist() == [len(t) for t in self.m.tables]
        for b, t in enumerate(self.m.tables):
            assert c.block_table[b, :len(t)].tolist() == t, b
        assert self.pool.refs.tolist() == self.m.refs()
        # every row a request has holds the bytes of the start row that the model has there
        at = [(p, k % 64) for b, n in enumerate(self.m.lens) for k in range(n) for p in [self.m.tables[b][k // 64]]]
        if not at:
            return
        page, slot = (torch.tensor(x, device=c.device) for x in zip(*at))
        tag = torch.from_numpy(self.m.tags).to(c.device)[page, slot]
        p0, s0 = tag // 64, tag % 64
        for layer, cache in enumerate(self.caches):
            if self.bits == 16:
                assert torch.equal(cache.pages.view(torch.int16)[page, slot], self.start[layer].view(torch.int16)[p0, s0])
                continue
            for lo, w in ((0, 512), (64 * 512, 64)):
                now, was = (t[:, lo:lo + 64 * w].unflatten(1, (64, w)) for t in (cache.pages, self.start[layer]))
                assert torch.equal(now[page, slot], was[p0, s0])
            assert torch.equal(cache.scales[page, slot // 16], self.scales[layer][p0, s0 // 16])


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("layers", [1, 3])
def test_operations_follow_the_model(cuda_device, bits, layers):
    """A long random sequence of operations; the state equals the model's after each."""
    rows = [0, 1, 63, 64, 65, 128, 200, 17]
    t = Twin(cuda_device, bits, layers, 8, 61, 6, rows)
    r = random.Random(bits + layers)
    t.check()
    for step in range(14):
        op = r.choice(("fork", "fork", "release", "reserve", "compact"))
        if op == "fork":
            dst = r.sample(range(8), r.randint(1, 8))
            src = [r.randrange(8) for _ in dst]
            if not t.m.fork(src, dst):
                with pytest.raises(native.MlaError):
                    t.pool.fork(src, dst, check="sync")
            else:
                t.pool.fork(src, dst, check="sync")
        elif op == "release":
            some = r.sample(range(8), r.randint(0, 2))
            t.m.release(some)
            t.pool.release(some, check="sync")
        elif op == "reserve":
            some = r.sample(range(8), r.randint(1, 8))
            n = r.randint(0, 100)
            if t.m.reserve(n, some):
                t.pool.reserve(n, some, check="sync")
        else:
            t.m.compact()
            t.pool.compact(check="sync")
        t.check()


@pytest.mark.parametrize("rows", [0, 1, 64, 65, 127, 128])
def test_fork_lengths(cuda_device, rows):
    t = Twin(cuda_device, 8, 2, 4, 20, 4, [rows, 0, 70, 3])
    t.m.fork([0, 0, 2], [1, 3, 2])
    t.pool.fork([0, 0, 2], [1, 3, 2], check="sync")
    t.check()


def test_many_requests_and_a_large_pool(cuda_device):
    """More pairs and pages than the planner's threads and step hold at once."""
    batch, n_pages = 1500, 40000
    table = torch.zeros(batch, 3, dtype=torch.int32, device=cuda_device)
    g = torch.Generator().manual_seed(0)
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    lens = torch.randint(0, 190, (batch,), generator=g).to(torch.int32)
    held = (lens + 63) // 64
    for b in range(batch):
        table[b, :held[b]] = order[3 * b:3 * b + int(held[b])]
    cache = fleet.PagedLatentCache8(n_pages, batch, 3, device=cuda_device, zero=False)
    cache.block_table.copy_(table)
    cache.seq_lens.copy_(lens)
    pool = fleet.PagePool(cache)
    src = torch.randperm(batch, generator=g).to(torch.int32)
    before, t0, refs0 = lens.clone(), table.cpu(), pool.refs.cpu()
    free = torch.nonzero(refs0 == 0)[:, 0].tolist()
    pool.fork(src.to(cuda_device), torch.arange(batch, dtype=torch.int32, device=cuda_device), check="sync")
    got, at = cache.block_table.cpu(), 0
    for b in range(batch):
        a = int(src[b])
        full, part = divmod(int(before[a]), 64)
        if a != b:
            assert got[b, :full].tolist() == t0[a, :full].tolist()
            if part:
                assert int(got[b, full]) == free[at]
                at += 1
    assert cache.seq_lens.cpu().tolist() == before[src.long()].tolist()
    h = pool.held.cpu()
    count = torch.bincount(torch.cat([got[b, :int(h[b])] for b in range(batch)]).long(), minlength=n_pages)
    assert torch.equal(count.to(torch.int32), pool.refs.cpu())
    live = int((pool.refs > 0).sum())
    pool.compact(check="sync")
    assert int((pool.refs[:live] > 0).sum()) == live
    pool.release(torch.arange(batch, dtype=torch.int32, device=cuda_device), check="sync")
    assert pool.free_pages() == n_pages
    cache.seq_lens.fill_(64)
    pool.reserve(1, check="sync")
    assert cache.block_table[:, :2].flatten().tolist() == list(range(2 * batch))


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n", [0, 1, 7, 400])
def test_copy_pages(cuda_device, bits, n):
    g = torch.Generator(device=cuda_device).manual_seed(n)
    def cache(pages):
        bt, sl = torch.zeros(1, 1, dtype=torch.int32, device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
        if bits == 16:
            return fleet.PagedLatentCache.from_tensors(torch.randn(pages, 64, 576, generator=g, device=cuda_device).to(BF), bt, sl)
        return fleet.PagedLatentCache8.from_tensors(
            torch.randint(0, 256, (pages, 36864), generator=g, device=cuda_device).to(torch.uint8),
            torch.randint(-64, 64, (pages, 4, 2), generator=g, device=cuda_device).to(torch.int8), bt, sl)
    a, b = [cache(500) for _ in range(2)], [cache(900) for _ in range(2)]
    src = torch.randperm(500, generator=g, device=cuda_device)[:n].to(torch.int32)
    dst = torch.randperm(900, generator=g, device=cuda_device)[:n].to(torch.int32)
    want = [c.pages.clone() for c in b]
    for w, c in zip(want, a):
        w[dst.long()] = c.pages[src.long()]
    fleet.copy_pages(a, src, b, dst)
    for w, c in zip(want, b):
        assert torch.equal(w.view(torch.uint8), c.pages.view(torch.uint8))
    if bits == 8 and n:
        assert torch.equal(b[1].scales[dst.long()], a[1].scales[src.long()])
    word = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    if n > 1:
        src[0], dst[1] = 500, -1
        fleet.copy_pages(a, src, b, dst, error_word=word)
        assert int(word) == 1


def test_errors_change_nothing(cuda_device):
    t = Twin(cuda_device, 8, 1, 4, 6, 4, [65, 64, 100, 0])  # 5 of 6 pages held
    for call, code in ((lambda: t.pool.fork([0, 2], [1, 3], check="sync"), 5),      # two pages wanted, one free
                       (lambda: t.pool.fork([0], [9], check="sync"), 6),
                       (lambda: t.pool.release([-1], check="sync"), 6),
                       (lambda: t.pool.reserve(300, [0], check="sync"), 2),         # past the block table
                       (lambda: t.pool.reserve(64, check="sync"), 5),
                       (lambda: t.pool.reserve(1, [7], check="sync"), 6)):
        with pytest.raises(native.MlaError) as e:
            call()
        assert e.value.code == code
        t.check()
    t.caches[0].seq_lens[0] = 200  # more rows than pages held
    t.m.lens[0] = 200
    with pytest.raises(native.MlaError) as e:
        t.pool.fork([0], [3], check="sync")
    assert e.value.code == 2


def test_refusals(cuda_device):
    c = fleet.PagedLatentCache8(4, 2, 2, device=cuda_device)
    d = fleet.PagedLatentCache8(4, 2, 2, device=cuda_device)
    e = fleet.PagedLatentCache(4, 2, 2, device=cuda_device)
    for caches in ([], [c, d], [c] * 65, [c, e]):
        with pytest.raises(ValueError):
            fleet.PagePool(caches)
    with pytest.raises(RuntimeError):
        fleet.PagePool(fleet.PagedLatentCache8(4, 2, 2, device="cpu"))
    pool = fleet.PagePool(c)
    with pytest.raises(ValueError):
        pool.fork([0], [1, 0])
    with pytest.raises(ValueError):
        pool.fork(torch.zeros(2, 2, dtype=torch.int32, device=cuda_device), [0])
    with pytest.raises(native.MlaError):
        pool.reserve(-1)
    with pytest.raises(native.MlaError):
        pool.fork([0, 0, 0], [1, 1, 1])  # more pairs than requests
    with pytest.raises(ValueError):
        fleet.copy_pages(c, [0], e, [1])
    with pytest.raises(ValueError):
        fleet.PagePool(c, held=torch.zeros(3, dtype=torch.int32, device=cuda_device))
    p, n = pool._p, pool.lib
    p.scratch_bytes -= 256
    assert n.mla_pool_compact(p, None) == -4
    p.scratch_bytes += 256
    p.scales[0] = 0
    assert n.mla_pool_compact(p, None) == -1
    p.scales[0] = c.scales.data_ptr() + 1
    assert n.mla_pool_compact(p, None) == -3


@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
def test_parallel_samples_decode_as_if_alone(cuda_device, window, sinks):
    """One prompt, forked into four samples that decode on, pages reserved, compacted and released on
    the way: each sample's outputs equal, bit for bit, those of a cache that it has to itself."""
    dev, n0, steps = cuda_device, 150, 30
    st = Step(dev, [n0], 500, window=window, sinks=sinks, max_pos=400)
    cache = fleet.PagedLatentCache8(40, 4, 8, device=dev)
    pool = fleet.PagePool(cache)
    prompt = random_rows(n0, 501).to(dev)
    cache.seq_lens[0] = n0
    pool.reserve(0, [0])
    fleet.rows_to_pages(cache, prompt, [0, n0, n0, n0, n0], [0, n0, n0, n0])
    pool.fork([0, 0, 0], [1, 2, 3])
    alone = []
    for _ in range(4):
        c = fleet.PagedLatentCache8.for_lengths([n0], extra_tokens=steps, device=dev)
        fleet.rows_to_pages(c, prompt, [0, n0], [0])
        alone.append(c)
    g = torch.Generator().manual_seed(502)
    for step in range(steps):
        q = torch.randn(4, 3072, generator=g).to(BF).to(dev)
        kv = torch.randn(4, 576, generator=g).to(BF).to(dev)
        pool.reserve(1)
        if step == 9:
            pool.compact(check="sync")
        out = st.runner.attend(q, kv, cache)
        cache.advance()
        for b in range(4):
            want = st.runner.attend(q[b:b + 1], kv[b:b + 1], alone[b], check="sync")
            # another split of the rows over CTAs: the same row values, sums in another order
            off = (out[b].float() - want[0].float()).norm() / want.float().norm()
            assert off <= 2.0 ** -8, (step, b)
            alone[b].advance()
    for b in range(4):
        n = n0 + steps
        assert torch.equal(cache.read_rows(b, 0, n), alone[b].read_rows(0, 0, n))
    pool.release([0, 1, 2, 3], check="sync")
    assert pool.free_pages() == 40


def test_operations_in_a_graph(cuda_device):
    """reserve + step + advance and a beam reorder, captured once and replayed."""
    dev = cuda_device
    st = Step(dev, [100], 510, max_pos=300)
    def make():
        cache = fleet.PagedLatentCache(30, 3, 5, device=dev)
        pool = fleet.PagePool(cache)
        cache.seq_lens.fill_(100)
        pool.reserve(0)
        for b in range(3):
            cache.write_rows(b, 0, random_rows(100, 511 + b))
        return cache, pool
    g = torch.Generator().manual_seed(512)
    q, kv = torch.randn(3, 3072, generator=g).to(BF).to(dev), torch.randn(3, 576, generator=g).to(BF).to(dev)
    src = torch.tensor([1, 0, 1], dtype=torch.int32, device=dev)
    dst = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    def step(cache, pool, out):
        pool.reserve(1)
        st.runner.attend(q, kv, cache, out)
        cache.advance()
        pool.fork(src, dst)
    a, pa = make()
    b, pb = make()
    oa, ob = torch.empty(3, 2048, dtype=BF, device=dev), torch.empty(3, 2048, dtype=BF, device=dev)
    step(a, pa, oa)
    step(b, pb, ob)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b, pb, ob)
    for _ in range(6):
        step(a, pa, oa)
        graph.replay()
        assert torch.equal(oa, ob)
    pa.raise_pending()
    pb.raise_pending()
    assert torch.equal(a.seq_lens, b.seq_lens) and torch.equal(pa.held, pb.held)
    for x in range(3):
        n = int(a.seq_lens[x])
        assert torch.equal(a.read_rows(x, 0, n), b.read_rows(x, 0, n))


@pytest.mark.parametrize("bits", [8, 16])
def test_a_step_on_a_released_request_stores_nothing(cuda_device, bits):
    """Its former page has gone to another request: the step reports the missing page and the new owner's
    rows stay as they are; after a reservation the request starts over."""
    dev = cuda_device
    st = Step(dev, [64, 0], 520, max_pos=300)
    cls = fleet.PagedLatentCache8 if bits == 8 else fleet.PagedLatentCache
    cache = cls(6, 2, 4, device=dev)
    pool = fleet.PagePool(cache)
    cache.seq_lens[0] = 64
    pool.reserve(1, [0])
    pool.release([0], check="sync")
    assert cache.block_table[0].tolist()[:2] == [-1, -1]
    cache.seq_lens[1] = 64
    pool.reserve(0, [1], check="sync")  # page 0, formerly request 0's
    rows = random_rows(64, 521).to(dev)
    fleet.rows_to_pages(cache, rows, [0, 0, 64])
    before = cache.read_rows(1, 0, 64).clone()
    pool.reserve(1, [1], check="sync")
    with pytest.raises(native.MlaError) as e:
        st.runner.attend(st.q, st.kv_a, cache, check="sync")
    assert e.value.code == 1
    assert torch.equal(cache.read_rows(1, 0, 64), before)
    pool.reserve(1, [0], check="sync")
    st.runner.attend(st.q, st.kv_a, cache, check="sync")
    assert torch.equal(cache.read_rows(1, 0, 64), before)


@pytest.mark.parametrize("bits,window", [(8, 0), (8, 100), (16, 0)])
def test_parallel_decode_example(cuda_device, bits, window):
    """The example end to end: samples advance, half end, what is left holds the shared prompt and its own pages."""
    import importlib
    example = importlib.import_module("fleet-mi300x_b200.parallel_decode")
    got = example.run(layers=3, prompt=150, samples=4, steps=40, window=window, sinks=4 if window else 0, bits=bits)
    assert got["rows"][:2] == [190, 190] and got["pages_held"] < got["pages_unshared"] + 2
    assert torch.isfinite(got["h"][:2].float()).all()


def test_stack_with_shared_row_counts_advances_once(cuda_device):
    st = Step(cuda_device, [10], 600, max_pos=64)
    own = fleet.PagedLatentCache8.for_lengths([10], extra_tokens=5, device=cuda_device)
    other = fleet.PagedLatentCache8(own.n_pages, 1, own.max_blocks, device=cuda_device)
    caches = [own, fleet.PagedLatentCache8.from_tensors(other.pages, other.scales, own.block_table, own.seq_lens)]
    stack = fleet.LayerStackGraph([st.runner] * 2, caches, mode="slice", advance=True)
    stack.replay()
    stack.synchronize()
    assert own.seq_lens.tolist() == [11]


@pytest.mark.parametrize("bits", [8, 16])
def test_a_step_past_a_fork_without_a_page_stores_nothing(cuda_device, bits):
    """A destination that had more pages than it gets: the step that needs another page, not reserved,
    reports it, and the rows of the request that its former page went to stay as they are."""
    dev = cuda_device
    st = Step(dev, [64, 64, 64], 530, max_pos=300)
    cls = fleet.PagedLatentCache8 if bits == 8 else fleet.PagedLatentCache
    cache = cls(6, 3, 4, device=dev)
    pool = fleet.PagePool(cache)
    cache.seq_lens.copy_(torch.tensor([64, 130, 0], dtype=torch.int32))
    pool.reserve(0)                       # request 0 page 0, request 1 pages 1, 2, 3
    rows = random_rows(64, 531).to(dev)
    fleet.rows_to_pages(cache, rows, [0, 64, 64, 64])
    pool.fork([0], [1], check="sync")     # request 1 shares page 0; pages 1, 2, 3 are free
    assert cache.block_table[1].tolist() == [0, -1, -1, 0]
    cache.seq_lens[2] = 128
    pool.reserve(0, [2], check="sync")    # pages 1 and 2, formerly request 1's
    fleet.rows_to_pages(cache, random_rows(128, 532).to(dev), [0, 0, 0, 128])
    before = cache.read_rows(2, 0, 128).clone()
    pool.reserve(1, [0, 2], check="sync")
    with pytest.raises(native.MlaError) as e:
        st.runner.attend(st.q, st.kv_a, cache, check="sync")
    assert e.value.code == 1
    assert torch.equal(cache.read_rows(2, 0, 128), before)
    pool.reserve(1, [1], check="sync")
    st.runner.attend(st.q, st.kv_a, cache, check="sync")
    assert torch.equal(cache.read_rows(2, 0, 128), before)


def test_the_example_releases_half_of_its_samples(cuda_device):
    """What it prints: the released samples have no rows and hold no pages afterwards, the others
    share the prompt's full pages and have one of their own."""
    import importlib
    example = importlib.import_module("fleet-mi300x_b200.parallel_decode")
    got = example.run(layers=2, prompt=150, samples=4, steps=40)
    assert got["rows"] == [190, 190, 0, 0]
    assert got["pages_held"] == 2 + 2 and got["pages_unshared"] == 2 * 3
    assert got["h"].shape[0] == 2
    got = example.run(layers=2, prompt=150, samples=1, steps=10)
    assert got["rows"] == [160] and got["pages_held"] == 3


def last_named(ids):
    """Each request once, where it is named last."""
    return [b for i, b in enumerate(ids) if b not in ids[i + 1:]]


@pytest.mark.parametrize("bits", [8, 16])
def test_operations_on_requests_named_twice(cuda_device, bits):
    """A destination named twice takes its last pair, beside the error; release acts once, and reserve
    gives pages once, where a request is named last."""
    t = Twin(cuda_device, bits, 2, 8, 61, 6, [0, 1, 63, 64, 65, 128, 200, 17])
    r = random.Random(bits)
    twice = {"fork": 0, "release": 0, "reserve": 0}
    for step in range(24):
        op = ("fork", "reserve", "fork", "release")[step % 4]
        ids = [r.randrange(8) for _ in range(8 if op == "fork" else 5)]
        twice[op] += len(set(ids)) < len(ids)
        if op == "fork":
            src = [r.randrange(8) for _ in ids]
            enough = t.m.fork(src, ids)
            if len(set(ids)) < len(ids) or not enough:
                with pytest.raises(native.MlaError) as e:
                    t.pool.fork(src, ids, check="sync")
                assert e.value.code == (6 if len(set(ids)) < len(ids) else 5)
            else:
                t.pool.fork(src, ids, check="sync")
        elif op == "release":
            ids = ids[:2] + ids[:1]
            t.m.release(ids)
            t.pool.release(ids, check="sync")
        else:
            n = r.randint(0, 100)
            if t.m.reserve(n, last_named(ids)):
                t.pool.reserve(n, ids, check="sync")
        t.check()
    assert all(twice.values())


def test_many_pairs_named_twice(cuda_device):
    """More pairs than the planner's threads, each destination named twice, far apart and next to itself."""
    batch, n_pages = 3000, 10000
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(0, 130, (batch,), generator=g).to(torch.int32)
    table = torch.arange(2 * batch, dtype=torch.int32).view(batch, 2).clone()
    cache = fleet.PagedLatentCache8(n_pages, batch, 2, device=cuda_device)
    lens.clamp_(max=128)
    cache.block_table.copy_(table)
    cache.seq_lens.copy_(lens)
    pool = fleet.PagePool(cache)
    free = torch.nonzero(pool.refs == 0)[:, 0].tolist()
    dst = torch.cat([torch.randperm(batch // 2, generator=g), torch.randperm(batch // 2, generator=g)]).to(torch.int32)
    dst[1::2][:500] = dst[0::2][:500]
    src = torch.randint(0, batch, (batch,), generator=g).to(torch.int32)
    with pytest.raises(native.MlaError) as e:
        pool.fork(src.to(cuda_device), dst.to(cuda_device), check="sync")
    assert e.value.code == 6
    last = {int(b): i for i, b in enumerate(dst)}
    want_lens, at = lens.tolist(), 0
    want = [table[b, :-(-int(lens[b]) // 64)].tolist() for b in range(batch)]
    new = {}
    for i in range(batch):
        a, b = int(src[i]), int(dst[i])
        if last[b] != i or a == b:
            continue
        full, part = divmod(int(lens[a]), 64)
        new[b] = table[a, :full].tolist() + ([free[at]] if part else [])
        at += part > 0
        want_lens[b] = int(lens[a])
    for b, t in new.items():
        want[b] = t
    got, held = cache.block_table.tolist(), pool.held.tolist()
    assert cache.seq_lens.tolist() == want_lens
    assert [got[b][:held[b]] for b in range(batch)] == want
    refs = torch.bincount(torch.tensor([p for t in want for p in t]), minlength=n_pages)
    assert pool.refs.tolist() == refs.tolist()


@pytest.mark.parametrize("bits", [8, 16])
def test_shared_pages_give_the_bits_of_pages_of_ones_own(cuda_device, bits):
    """Four samples that share their prompt's full pages, and four that hold copies of them, in the same batch and
    so on the same split: equal outputs and rows, bit for bit."""
    dev, n0, steps = cuda_device, 150, 20
    st = Step(dev, [n0], 540, max_pos=400)
    cls = fleet.PagedLatentCache8 if bits == 8 else fleet.PagedLatentCache
    cache = cls(40, 4, 8, device=dev)
    pool = fleet.PagePool(cache)
    prompt = random_rows(n0, 541).to(dev)
    cache.seq_lens[0] = n0
    pool.reserve(0, [0])
    fleet.rows_to_pages(cache, prompt, [0] + [n0] * 4)
    pool.fork([0, 0, 0], [1, 2, 3])
    own = cls.for_lengths([n0] * 4, extra_tokens=steps, device=dev)
    fleet.rows_to_pages(own, prompt.repeat(4, 1), [n0 * b for b in range(5)])
    g = torch.Generator().manual_seed(542)
    for step in range(steps):
        q = torch.randn(4, 3072, generator=g).to(BF).to(dev)
        kv = torch.randn(4, 576, generator=g).to(BF).to(dev)
        pool.reserve(1)
        assert torch.equal(st.runner.attend(q, kv, cache, check="sync"), st.runner.attend(q, kv, own, check="sync")), step
        cache.advance()
        own.advance()
    for b in range(4):
        assert torch.equal(cache.read_rows(b, 0, n0 + steps), own.read_rows(b, 0, n0 + steps))
