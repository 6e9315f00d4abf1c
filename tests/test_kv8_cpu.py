"""The 8-bit cache without a GPU: its class, its refusals, the library's argument checks, and the
64-bit restatement that the GPU tests rely on, checked against torch's e4m3."""
import ctypes
import importlib

import numpy as np
import pytest
import torch

import kv8_testlib as R
from mla_testlib import fleet

native = importlib.import_module("fleet-mi300x_b200.native")


def test_cache_shapes_and_adoption():
    c = fleet.PagedLatentCache8(3, 2, 4, device="cpu")
    assert c.pages.shape == (3, 36864) and c.pages.dtype == torch.uint8
    assert c.scales.shape == (3, 4, 2) and c.scales.dtype == torch.int8
    assert (c.batch, c.n_pages, c.max_blocks) == (2, 3, 4)
    d = fleet.PagedLatentCache8.from_tensors(c.pages, c.scales, c.block_table, c.seq_lens)
    assert d.pages.data_ptr() == c.pages.data_ptr() and isinstance(d, fleet.PagedLatentCache)
    e = fleet.PagedLatentCache.from_tensors(torch.zeros(3, 64, 576, dtype=torch.bfloat16), c.block_table, c.seq_lens)
    assert e.n_pages == 3
    f = fleet.PagedLatentCache8.for_lengths([5, 64, 130], device="cpu")
    assert f.max_blocks == 3 and f.seq_lens.tolist() == [5, 64, 130]


@pytest.mark.parametrize("field,bad", [
    ("pages", lambda t: t[:, :-1]), ("pages", lambda t: t.to(torch.int16)), ("pages", lambda t: t[::2]),
    ("scales", lambda t: t[:2]), ("scales", lambda t: t.to(torch.int32)), ("block_table", lambda t: t.long()),
    ("seq_lens", lambda t: t[:1]), ("block_table", lambda t: t.t())])
def test_adoption_refuses(field, bad):
    c = fleet.PagedLatentCache8(4, 2, 4, device="cpu")
    kw = dict(pages=c.pages, scales=c.scales, block_table=c.block_table, seq_lens=c.seq_lens)
    kw[field] = bad(kw[field])
    with pytest.raises(ValueError):
        fleet.PagedLatentCache8.from_tensors(**kw)


def test_read_rows_decodes_pages_and_scales():
    c = fleet.PagedLatentCache8(2, 1, 2, device="cpu")
    c.block_table[0] = torch.tensor([1, 0])
    rng = np.random.RandomState(0)
    rows = R.bf16(rng.randn(100, 576))
    want = R.Cache8(100)
    want.write(0, rows)
    for t in range(100):
        pg, sl = int(c.block_table[0, t // 64]), t % 64
        code = torch.from_numpy(want.codes[t]).float().to(torch.float8_e4m3fn).view(torch.uint8)
        c.pages[pg, sl * 512:sl * 512 + 512] = code[:512]
        c.pages[pg, 32768 + sl * 64:32768 + sl * 64 + 64] = code[512:]
        c.scales[pg, sl // 16] = torch.from_numpy(want.exps[t // 16].astype(np.int8))
    got = c.read_rows(0, 0, 100).double().numpy()
    assert np.array_equal(got, want.values(100))
    # half of an e4m3 step (2^-4 of the value), or of the smallest step (2^-9) under the block's scale
    step = np.exp2(np.repeat(want.exps, 16, 0)[:100].astype(np.float64))
    step = np.concatenate([np.repeat(step[:, :1], 512, 1), np.repeat(step[:, 1:], 64, 1)], 1)
    assert (np.abs(got - rows) <= np.maximum(np.abs(rows) * 2.0 ** -4, step * 2.0 ** -10)).all()


def test_restatement_rounds_as_torch():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.randn(5000) * 0.01, torch.randn(5000) * 1e-3])
    assert np.array_equal(R.round_e4m3(x.double().numpy()), x.to(torch.float8_e4m3fn).double().numpy())
    y = torch.randn(10000) * torch.exp2(torch.linspace(-120, 120, 10000))
    assert np.array_equal(R.bf16(y.double().numpy()), y.to(torch.bfloat16).double().numpy())


def test_library_refuses_before_it_launches():
    lib = native.load_library()
    n = ctypes.c_uint64()
    p = native.new_params()
    p.batch, p.num_ctas, p.flags = 4, 8, native.FLAG_KV8
    assert lib.mla_workspace_size(ctypes.byref(p), ctypes.byref(n)) == 0
    assert lib.mla_decode_step(ctypes.byref(p), None) == -1  # null pointers
    r = native.new_rows()
    assert not r.kv_scales and lib.mla_rows_to_pages(ctypes.byref(r), None) == -1
