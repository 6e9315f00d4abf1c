"""The 8-bit latent cache and what a server does with it, as measurable cases.

Four operators of an absorbed multi-head latent attention (MLA) decoder: 16 heads, rows of
512 latent + 64 rotary columns, pages of 64 rows behind a block table.

  rows    finished bf16 rows of a prompt stored into the pages of an 8-bit cache
  attend  one decode step (append one row, attend over all rows) on the 8-bit cache
  window  the same with a sliding window and a few first rows that stay visible
  fork    requests that become copies of others: shared full pages, a copied last page
  copy    pages copied to other pages

The 8-bit cache: a page is 36,864 bytes, first the latent part [64][512], then the rotary part
[64][64], both e4m3. Each block of 16 rows of a page has one power-of-two scale per part, held as its
exponent: value = e4m3 * 2^exponent, with the smallest exponent (at least -64) that brings the
block's largest magnitude to at most 448. When a row joins a block whose scale is too small for it, the
block's earlier rows are held anew under the larger one.

`run` computes the operators in plain torch where `own` is false, and through the framework's
public entry points where it is true.
"""
import importlib
import math
import random

import torch

own = False

HEADS, NOPE, ROPE, V, LORA = 16, 128, 64, 128, 512
ROW = LORA + ROPE
PAGE, BLOCK = 64, 16
PAGE8 = PAGE * ROW
EPS = 1e-6
SCALE = (NOPE + ROPE) ** -0.5 * (0.1 * 0.707 * math.log(40.0) + 1.0) ** 2
F8 = torch.float8_e4m3fn
BF = torch.bfloat16
DEV = "cuda"


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # a short prompt's rows: latency of one call
        {"name": "rows_1x17", "op": "rows", "batch": 1, "lo": 17, "hi": 17, "first": 0},
        # chunks of a batched prefill, continued at odd positions, some requests without rows
        {"name": "rows_32_chunks", "op": "rows", "batch": 32, "lo": 0, "hi": 1024, "first": 2000},
        # one long prompt
        {"name": "rows_1x131072", "op": "rows", "batch": 1, "lo": 131072, "hi": 131072, "first": 0},
        # single layer, one request, a short context (the framework's config 1)
        {"name": "attend_1x1024", "op": "attend", "batch": 1, "lo": 1024, "hi": 1024},
        # ragged batch (config 3)
        {"name": "attend_32_ragged", "op": "attend", "batch": 32, "lo": 512, "hi": 8192},
        # a full decode batch (config 5a), the largest case
        {"name": "attend_256x4096", "op": "attend", "batch": 256, "lo": 4096, "hi": 4096},
        # one very long sequence (config 5b)
        {"name": "attend_1x131072", "op": "attend", "batch": 1, "lo": 131072, "hi": 131072},
        # streaming decode of one long conversation: 4 first rows and the last 4096, 8-bit cache
        {"name": "window_1_of_131072", "op": "window", "batch": 1, "lo": 131072, "hi": 131072, "window": 4096,
         "sinks": 4, "bits": 8},
        # a ragged batch under an odd window on the bf16 cache
        {"name": "window_32_bf16", "op": "window", "batch": 32, "lo": 512, "hi": 8192, "window": 1000, "sinks": 5,
         "bits": 16},
        # one prompt sampled four ways, 8-bit caches of all 27 layers
        {"name": "fork_4_of_1", "op": "fork", "batch": 4, "parents": 1, "rows": 1000, "layers": 27, "bits": 8},
        # beams reordered among themselves, bf16 caches of all layers
        {"name": "fork_64_beams", "op": "fork", "batch": 64, "parents": 64, "rows": 500, "layers": 27, "bits": 16},
        # pages moved to other places of a layer's pool
        {"name": "copy_2048_pages", "op": "copy", "pages": 2048, "bits": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rows", "attend", "attend", "window", "window", "fork", "copy"))
    if op == "rows":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, max(2, 131072 // batch))
        return {"op": op, "batch": batch, "lo": rng.randint(0, hi) if batch > 1 else hi, "hi": hi,
                "first": rng.choice((0, rng.randint(1, 300)))}
    if op in ("attend", "window"):
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, 1_000_000 // batch) if batch > 8 else _log(rng, 1, 131072)
        case = {"op": op, "batch": batch, "lo": rng.choice((hi, rng.randint(0, hi))), "hi": hi}
        if op == "window":
            case |= {"window": _log(rng, 1, 8192), "sinks": rng.choice((0, 1, 4, rng.randint(2, 200))),
                     "bits": rng.choice((8, 16))}
        return case
    if op == "fork":
        batch = _log(rng, 2, 64)
        return {"op": op, "batch": batch, "parents": rng.choice((1, rng.randint(1, batch), batch)),
                "rows": _log(rng, 1, 4000), "layers": rng.choice((1, rng.randint(2, 26), 27)),
                "bits": rng.choice((8, 16))}
    return {"op": op, "pages": _log(rng, 1, 4096), "bits": rng.choice((8, 16))}


# ---------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(case):
    """The requests' lengths, whole numbers in [lo, hi] and the first one hi: a case's own, whatever the seed."""
    r = random.Random(case["batch"] * 1_000_003 + case["hi"])
    return [case["hi"]] + [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"] - 1)]


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e, at least -64."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8).clamp_min(-64)
    return torch.where(amax > 0, e, torch.full_like(e, -64)).to(torch.int32)


def _pow2(e):
    return torch.exp2(e.to(torch.float32))


def _pool(n_pages, bits, g):
    """A layer's pool of pages with N(0, 1) rows: (pages, scales), scales None for bf16."""
    if bits == 16:
        return torch.randn(n_pages, PAGE, ROW, generator=g, device=DEV, dtype=torch.float32).to(BF) \
            if n_pages <= 8192 else torch.cat([_pool(min(8192, n_pages - i), 16, g)[0]
                                               for i in range(0, n_pages, 8192)]), None
    pages = torch.empty(n_pages, PAGE8, dtype=torch.uint8, device=DEV)
    scales = torch.empty(n_pages, PAGE // BLOCK, 2, dtype=torch.int8, device=DEV)
    for i in range(0, n_pages, 2048):
        n = min(2048, n_pages - i)
        x = torch.randn(n, PAGE, ROW, generator=g, device=DEV).to(BF).float().view(n, PAGE // BLOCK, BLOCK, ROW)
        for k, (a, b) in enumerate(((0, LORA), (LORA, ROW))):
            part = x[..., a:b]
            e = _exponent(part.abs().amax((2, 3)))
            q = (part * _pow2(-e)[:, :, None, None]).to(F8).view(torch.uint8)
            pages[i:i + n, PAGE * a:PAGE * b] = q.reshape(n, -1)
            scales[i:i + n, :, k] = e.to(torch.int8)
    return pages, scales


def _table(rows, g, spare=0):
    """A block table that gives each request the pages for its rows, in random order."""
    need = [max(1, -(-r // PAGE)) for r in rows]
    n = sum(need) + spare
    order = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(rows), max(need), dtype=torch.int32, device=DEV)
    starts = torch.tensor([0] + need[:-1], device=DEV).cumsum(0)
    need_d = torch.tensor(need, device=DEV)
    col = torch.arange(table.shape[1], device=DEV)
    inside = col[None, :] < need_d[:, None]
    table[inside] = order[(starts[:, None] + col[None, :])[inside]]
    return table, n


def _rope_tables(n):
    f = 1.0 / (10000.0 ** (torch.arange(0, ROPE, 2, device=DEV, dtype=torch.float64) / ROPE))
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * torch.cat([f, f])[None, :]
    return a.cos().float(), a.sin().float()


def _inputs(case, seed):
    """The tensors of a case, from its seed alone."""
    g = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op == "rows":
        n = _lengths(case)
        first = [case["first"] + 7 * (b % 3) if case["first"] else 0 for b in range(case["batch"])]
        s["table"], s["n_pages"] = _table([a + b for a, b in zip(n, first)], g)
        s["pages"], s["scales"] = _pool(s["n_pages"], 8, g)
        s["row_start"] = torch.tensor([0] + n, device=DEV).cumsum(0)
        s["first"] = torch.tensor(first, dtype=torch.int32, device=DEV)
        s["total"] = sum(n)
        s["rows"] = torch.randn(max(1, sum(n)), ROW, generator=g, device=DEV).to(BF)[:sum(n)]
        s["lens"] = s["first"].clone()
    elif op in ("attend", "window"):
        n = _lengths(case)
        B = case["batch"]
        s["table"], s["n_pages"] = _table([x + 1 for x in n], g)
        s["pages"], s["scales"] = _pool(s["n_pages"], case.get("bits", 8), g)
        s["lens"] = torch.tensor(n, dtype=torch.int32, device=DEV)
        s["cos"], s["sin"] = _rope_tables(max(n) + 1)
        x = torch.randn(B, 2048, generator=g, device=DEV)
        w = torch.randn(HEADS * (NOPE + ROPE) + ROW, 2048, generator=g, device=DEV) * 0.02
        qkv = (x @ w.T).to(BF)
        s["q"], s["kv_a"] = qkv[:, :HEADS * (NOPE + ROPE)], qkv[:, HEADS * (NOPE + ROPE):]
        s["norm"] = (torch.rand(LORA, generator=g, device=DEV) * 0.4 + 0.8).to(BF)
        s["kv_b"] = (torch.randn(HEADS * (NOPE + V), LORA, generator=g, device=DEV) * 0.02).to(BF)
    elif op == "fork":
        B, L = case["batch"], case["layers"]
        rows = [case["rows"] if b < case["parents"] else 0 for b in range(B)]
        s["table"], s["n_pages"] = _table([case["rows"]] * B, g, spare=B + 3)
        held = torch.tensor([-(-r // PAGE) for r in rows], dtype=torch.int32, device=DEV)
        s["held"], s["lens"] = held, torch.tensor(rows, dtype=torch.int32, device=DEV)
        inside = torch.arange(s["table"].shape[1], device=DEV)[None, :] < held[:, None]
        s["refs"] = torch.zeros(s["n_pages"], dtype=torch.int32, device=DEV)
        s["refs"][s["table"][inside].long()] = 1
        pages, scales = _pool(s["n_pages"] * L, case["bits"], g)
        s["pages"] = pages.view(L, s["n_pages"], *pages.shape[1:])
        s["scales"] = None if scales is None else scales.view(L, s["n_pages"], PAGE // BLOCK, 2)
        # one pass: every request but the first takes over the state of a parent
        s["dst"] = torch.arange(1, B, dtype=torch.int32, device=DEV)
        s["src"] = torch.randint(0, case["parents"], (B - 1,), generator=g, device=DEV).to(torch.int32)
    else:
        n = case["pages"]
        s["n_pages"] = 2 * n + 1
        s["pages"], s["scales"] = _pool(s["n_pages"], case["bits"], g)
        order = torch.randperm(s["n_pages"], generator=g, device=DEV).to(torch.int32)
        s["src"], s["dst"] = order[:n].contiguous(), order[n:2 * n].contiguous()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        P = importlib.import_module("fleet-mi300x_b200")
        op = case["op"]
        wrap = (lambda pg, sc, t, n: P.PagedLatentCache.from_tensors(pg, t, n)) if case.get("bits", 8) == 16 else \
            P.PagedLatentCache8.from_tensors
        if op == "fork":
            caches = [wrap(s["pages"][k], None if s["scales"] is None else s["scales"][k], s["table"], s["lens"])
                      for k in range(case["layers"])]
            s["pool"] = P.PagePool(caches, held=s["held"], refs=s["refs"])
        elif op == "copy":
            s["cache"] = wrap(s["pages"], s["scales"], torch.zeros(1, 1, dtype=torch.int32, device=DEV),
                              torch.zeros(1, dtype=torch.int32, device=DEV))
        else:
            s["cache"] = wrap(s["pages"], s["scales"], s["table"], s["lens"])
        if op in ("attend", "window"):
            w = P.LayerWeights(torch.zeros(HEADS * (NOPE + ROPE), 2048, dtype=BF, device=DEV),
                               torch.zeros(ROW, 2048, dtype=BF, device=DEV), s["norm"], s["kv_b"])
            s["runner"] = P.MlaDecodeAttention(P.ModelConfig(), w, s["cos"], s["sin"],
                                               window=case.get("window", 0), sinks=case.get("sinks", 0))
        s["lib"] = P
    return s


# ---------------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        P = s["lib"]
        if op == "rows":
            P.rows_to_pages(s["cache"], s["rows"], s["row_start"], s["first"], total=s["total"])
        elif op in ("attend", "window"):
            return _state(s) | {"out": s["runner"].attend(s["q"], s["kv_a"], s["cache"])}
        elif op == "fork":
            s["pool"].fork(s["src"], s["dst"])
        else:
            P.copy_pages(s["cache"], s["src"], s["cache"], s["dst"])
        return _state(s)
    if op == "rows":
        _plain_rows(s)
    elif op in ("attend", "window"):
        return _state(s) | {"out": _plain_attend(s)}
    elif op == "fork":
        _plain_fork(s)
    else:
        s["pages"][s["dst"].long()] = s["pages"][s["src"].long()]
        if s["scales"] is not None:
            s["scales"][s["dst"].long()] = s["scales"][s["src"].long()]
    return _state(s)


def _state(s):
    """What a pass leaves in the caches: 8-bit pages as the e4m3 values that their bytes are."""
    got = {"pages": s["pages"] if s["scales"] is None else s["pages"].view(F8)}
    for k in ("scales",) if s["case"]["op"] != "fork" else ("scales", "table", "lens", "held", "refs"):
        if s[k] is not None:
            got[k] = s[k]
    return got


# ---------------------------------------------------------------------------------- plain forms
def _parts(pages):
    """The two parts of 8-bit pages [n, 36864] as e4m3 [n, 4, 16, columns] views."""
    p = pages.view(F8)
    return (p[:, :PAGE * LORA].view(-1, PAGE // BLOCK, BLOCK, LORA),
            p[:, PAGE * LORA:].view(-1, PAGE // BLOCK, BLOCK, ROPE))


def _store8(s, rows, page, slot, first_page, first_slot, joins):
    """Rows [n, 576] into (page, slot); `joins` [b]: the block of (first_page, first_slot) has
    earlier rows, which share its scale."""
    n_pages = s["pages"].shape[0]
    block = page * (PAGE // BLOCK) + slot // BLOCK
    head = first_page * (PAGE // BLOCK) + first_slot // BLOCK
    inner = torch.arange(BLOCK, device=DEV)
    for k, (a, b) in enumerate(((0, LORA), (LORA, ROW))):
        x = rows[:, a:b].float()
        amax = torch.zeros(n_pages * (PAGE // BLOCK), device=DEV).scatter_reduce(0, block, x.abs().amax(1), "amax")
        e = _exponent(amax)
        old = s["scales"].view(-1, 2)[:, k].to(torch.int32)
        e_head = torch.where(joins, torch.maximum(e[head], old[head]), e[head])
        e[head] = e_head
        codes = _parts(s["pages"])[k]
        # the earlier rows of a joined block, held anew under its scale
        at = (first_page, first_slot // BLOCK)
        was = codes[at].float() * _pow2(old[head] - e_head)[:, None, None]
        keep = joins[:, None] & (inner[None, :] < (first_slot % BLOCK)[:, None])
        raw = codes.view(torch.uint8)
        raw[at] = torch.where(keep[:, :, None], was.to(F8).view(torch.uint8), raw[at])
        raw[page, slot // BLOCK, slot % BLOCK] = (x * _pow2(-e[block])[:, None]).to(F8).view(torch.uint8)
        s["scales"].view(-1, 2)[block, k] = e[block].to(torch.int8)


def _plain_rows(s):
    i = torch.arange(s["total"], device=DEV)
    b = torch.searchsorted(s["row_start"], i, right=True) - 1
    pos = s["first"][b] + i - s["row_start"][b]
    page = s["table"][b, pos // PAGE].long()
    some = s["row_start"][1:] > s["row_start"][:-1]
    first = s["first"].long()[some]
    _store8(s, s["rows"], page, pos % PAGE, s["table"][some].gather(1, first[:, None] // PAGE)[:, 0].long(),
            first % PAGE, first % BLOCK > 0)


def _rope(x, cos, sin):
    """x [..., 64] in interleaved pairs, rotated; the halves of the result hold the pairs' two sides."""
    even, odd = x[..., 0::2], x[..., 1::2]
    h = ROPE // 2
    return torch.cat([even * cos[..., :h] - odd * sin[..., :h], odd * cos[..., h:] + even * sin[..., h:]], -1)


def _plain_attend(s):
    B, n = s["case"]["batch"], s["lens"].long()
    window, sinks = s["case"].get("window", 0), s["case"].get("sinks", 0)
    cos, sin = s["cos"][n], s["sin"][n]
    # the new row: the model's own bf16 row (norm, weight and rotation each rounded), appended at row n
    kv = s["kv_a"].float()
    c = kv[:, :LORA]
    c = (c / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)).to(BF).float() * s["norm"].float()
    row = torch.cat([c, _rope(kv[:, LORA:], cos, sin)], 1).to(BF)
    page = s["table"].gather(1, n[:, None] // PAGE)[:, 0].long()
    if s["scales"] is None:
        s["pages"][page, n % PAGE] = row
    else:
        _store8(s, row, page, n % PAGE, page, n % PAGE, n % BLOCK > 0)
    # absorbed query
    q = s["q"].float().view(B, HEADS, NOPE + ROPE)
    w = s["kv_b"].float().view(HEADS, NOPE + V, LORA)
    qa = torch.cat([torch.einsum("bhd,hdc->bhc", q[..., :NOPE], w[:, :NOPE]),
                    _rope(q[..., NOPE:], cos[:, None], sin[:, None])], -1)
    # the visible rows of every request, padded to the most that one has
    most = s["case"]["hi"] + 1
    if window and window + sinks < most:
        j = torch.arange(sinks + window, device=DEV)[None, :]
        from_ = (n + 1 - window).clamp_min(0)[:, None]
        t = torch.where(j < sinks, j, j - sinks + from_)
        seen = (t <= n[:, None]) & ((j < sinks) | (t >= sinks))
        t = t.clamp_max(most - 1)
    else:
        t = torch.arange(most, device=DEV)[None, :].expand(B, -1)
        seen = t <= n[:, None]
        if window:
            seen = seen & ((t < sinks) | (t > n[:, None] - window))
    at = s["table"].gather(1, (t // PAGE)).long()
    if s["scales"] is None:
        k = s["pages"][at, t % PAGE].float()
    else:
        f = _pow2(s["scales"][at, t % PAGE // BLOCK])
        k = torch.cat([x[at, t % PAGE // BLOCK, t % BLOCK].float() * f[..., j:j + 1]
                       for j, x in enumerate(_parts(s["pages"]))], -1)
    x = torch.matmul(qa, k.transpose(1, 2)) * SCALE
    x = torch.where(seen[:, None, :], x, torch.full_like(x, float("-inf")))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(x / x.sum(-1, keepdim=True), k[..., :LORA])
    return torch.einsum("bhc,hvc->bhv", o, w[:, NOPE:]).reshape(B, HEADS * V).to(BF)


def _plain_fork(s):
    src, dst, table, held, lens, refs = (s[k] for k in ("src", "dst", "table", "held", "lens", "refs"))
    moves = src != dst
    src, dst = src[moves].long(), dst[moves].long()
    rows = lens[src].long()
    full, part = rows // PAGE, rows % PAGE
    # a page of its own for every last page that is not full: the lowest free ones, in order
    need = part > 0
    free = torch.nonzero(refs == 0)[:, 0]
    fresh = free[(need.long().cumsum(0) - 1).clamp_min(0)]
    col = torch.arange(table.shape[1], device=DEV)[None, :]
    old = table[dst]
    drop = old[col < held[dst][:, None]].long()
    from_ = table[src]
    share = from_[col < full[:, None]].long()
    new = torch.where(col < full[:, None], from_, old)
    new = torch.where((col == full[:, None]) & need[:, None], fresh[:, None].to(torch.int32), new)
    refs.scatter_add_(0, share, torch.ones_like(share, dtype=torch.int32))
    refs.scatter_add_(0, drop, torch.full_like(drop, -1, dtype=torch.int32))
    refs[fresh[need]] = 1
    # the rows of those last pages, in every layer
    last = from_.gather(1, full.clamp_max(table.shape[1] - 1)[:, None])[:, 0].long()[need]
    to, here = fresh[need], torch.arange(PAGE, device=DEV)[None, :] < part[need][:, None]
    if s["scales"] is None:
        s["pages"][:, to] = torch.where(here[None, :, :, None], s["pages"][:, last], s["pages"][:, to])
    else:
        L, n = s["pages"].shape[:2]
        both = _parts(s["pages"].view(L * n, PAGE8))
        blocks = here.view(-1, PAGE // BLOCK, BLOCK, 1)
        for p in both:
            v = p.view(torch.uint8).unflatten(0, (L, n))
            v[:, to] = torch.where(blocks, v[:, last], v[:, to])
        s["scales"][:, to] = s["scales"][:, last]
    table[dst] = new
    held[dst] = (full + need).to(torch.int32)
    lens[dst] = rows.to(torch.int32)


# ---------------------------------------------------------------------------------- work, 64-bit values
def _seen(n, window, sinks):
    """How many rows a query at row n sees."""
    return n + 1 if not window or n + 1 <= window else window + min(sinks, n + 1 - window)


def work(case):
    op, bits = case["op"], case.get("bits", 8)
    row = ROW * bits // 8 + (2 / BLOCK if bits == 8 else 0)
    if op == "rows":
        n = sum(_lengths(case))
        return {"bytes": max(1.0, n * (2 * ROW + row)), "flops": 3.0 * ROW * n}
    if op in ("attend", "window"):
        B = case["batch"]
        seen = sum(_seen(n, case.get("window", 0), case.get("sinks", 0)) for n in _lengths(case))
        per = HEADS * (NOPE + ROPE) * 2 + ROW * 2 + row + HEADS * V * 2
        return {"bytes": seen * row + B * per + 2.0 * HEADS * (NOPE + V) * LORA,
                "flops": seen * 2.0 * HEADS * (ROW + LORA) + B * 4.0 * HEADS * NOPE * LORA}
    if op == "fork":
        part, full = case["rows"] % PAGE, case["rows"] // PAGE
        moved = (case["batch"] - 1) * (1 - (1 / case["parents"] if case["parents"] > 1 else 0))
        return {"bytes": max(64.0, moved * (2 * case["layers"] * part * row + 20 * (full + 1))), "flops": 0.0}
    return {"bytes": 2.0 * case["pages"] * PAGE * row, "flops": 0.0}


def _round_e4m3(x):
    """x to the nearest e4m3 value, ties to even, in 64 bits (|x| <= 448)."""
    e = (torch.frexp(x.abs())[1] - 1).clamp_min(-6)
    step = torch.exp2(e.double() - 3)
    return torch.round(x / step) * step


def _smallest_exponent(a):
    e = -64
    while a > 448.0 * 2.0 ** e:
        e += 1
    return e


class _Exact8:
    """An 8-bit cache as 64-bit codes of the rows that a case touches."""

    def __init__(self, s):
        self.p = s["pages"].view(F8)
        self.e = s["scales"].double()

    def codes(self, pages):
        p = self.p[pages].to(torch.float64)
        return torch.cat([p[:, :PAGE * LORA].view(-1, PAGE, LORA), p[:, PAGE * LORA:].view(-1, PAGE, ROPE)], 2)

    def values(self, pages):
        """[n, 64, 576] of the pages."""
        f = torch.exp2(self.e[pages]).repeat_interleave(BLOCK, 1)
        return self.codes(pages) * torch.cat([f[..., :1].expand(-1, -1, LORA), f[..., 1:].expand(-1, -1, ROPE)], 2)


def _join(before, exps, row):
    """A block's earlier codes [m, 576] under exponents exps (2), and a row [576] that joins it:
    the values of all m + 1 rows."""
    got = []
    for k, (a, b) in enumerate(((0, LORA), (LORA, ROW))):
        e = _smallest_exponent(float(row[a:b].abs().max()))
        if before.shape[0]:
            e = max(e, int(exps[k]))
        old = _round_e4m3(before[:, a:b] * 2.0 ** (int(exps[k]) - e))
        got.append(torch.cat([old, _round_e4m3(row[None, a:b] * 2.0 ** -e)]) * 2.0 ** e)
    return torch.cat(got, 1)


def exact(case, seed):
    op = case["op"]
    if op == "fork" or op == "copy":
        return None  # nothing is computed: bytes that move
    s = _inputs(case, seed)
    if op == "rows":
        return _exact_rows(s)
    bits, window, sinks = case.get("bits", 8), case.get("window", 0), case.get("sinks", 0)
    cache = _Exact8(s) if bits == 8 else None
    W = s["kv_b"].double().view(HEADS, NOPE + V, LORA)
    norm, cos, sin = s["norm"].double(), s["cos"].double(), s["sin"].double()
    out = torch.empty(case["batch"], HEADS * V, dtype=torch.float64, device=DEV)

    def turn(x, n):
        y = torch.empty_like(x)
        y[..., :32] = x[..., 0::2] * cos[n, :32] - x[..., 1::2] * sin[n, :32]
        y[..., 32:] = x[..., 1::2] * cos[n, 32:] + x[..., 0::2] * sin[n, 32:]
        return y

    for b, n in enumerate(s["lens"].tolist()):
        kv = s["kv_a"][b].double()
        c = kv[:LORA] * (kv[:LORA].square().mean() + EPS).rsqrt()
        new = torch.cat([(c.to(BF).double() * norm).to(BF).double(), turn(kv[LORA:], n).to(BF).double()])
        first = max(0, n + 1 - window) if window else 0
        head = min(sinks, first) if window else 0
        t = torch.cat([torch.arange(head, device=DEV), torch.arange(first, n, device=DEV)])
        page = s["table"][b].long()
        if bits == 16:
            rows = torch.cat([s["pages"][page[t // PAGE], t % PAGE].double(), new[None]])
        else:
            used, where = torch.unique(t // PAGE, return_inverse=True)
            rows = cache.values(page[used])[where, t % PAGE] if t.numel() else new.new_empty(0, ROW)
            own_page, lo = page[n // PAGE], n % PAGE // BLOCK * BLOCK
            block = _join(cache.codes(own_page[None])[0, lo:n % PAGE], cache.e[own_page, lo // BLOCK].tolist(), new)
            start = n // BLOCK * BLOCK
            again = (t >= start).nonzero()[:, 0]
            rows[again] = block[t[again] - start]
            rows = torch.cat([rows, block[-1:]])
        q = s["q"][b].double().view(HEADS, NOPE + ROPE)
        qa = torch.cat([torch.bmm(q[:, None, :NOPE], W[:, :NOPE])[:, 0], turn(q[:, NOPE:], n)], 1)
        p = torch.softmax(qa @ rows.T * SCALE, 1)
        o = p @ rows[:, :LORA]
        out[b] = torch.bmm(W[:, NOPE:], o[:, :, None]).reshape(-1)
    return {"pages": None, "scales": None, "out": out} if bits == 8 else {"pages": None, "out": out}


def _exact_rows(s):
    """The codes of all pages after the rows were stored, in the pages' order."""
    p = s["pages"].view(F8).double()
    c = p[:, :PAGE * LORA].reshape(-1, PAGE, LORA)
    r = p[:, PAGE * LORA:].reshape(-1, PAGE, ROPE)
    starts, firsts = s["row_start"].tolist(), s["first"].tolist()
    for b, first in enumerate(firsts):
        rows = s["rows"][starts[b]:starts[b + 1]].double()
        n = rows.shape[0]
        if not n:
            continue
        pos = torch.arange(first, first + n, device=DEV)
        page, slot = s["table"][b].long()[pos // PAGE], pos % PAGE
        nth = pos // BLOCK - first // BLOCK
        for k, (a, z, to) in enumerate(((0, LORA, c), (LORA, ROW, r))):
            top = torch.zeros(int(nth[-1]) + 1, dtype=torch.float64, device=DEV)
            top.scatter_reduce_(0, nth, rows[:, a:z].abs().amax(1), "amax")
            e = torch.ceil(torch.log2(top / 448.0)).clamp_min(-64)
            e = torch.where(448.0 * torch.exp2(e - 1) >= top, e - 1, e).clamp_min(-64)
            e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
            e = torch.where(top > 0, e, torch.full_like(e, -64.0))
            if first % BLOCK:
                was = float(s["scales"][page[0], slot[0] // BLOCK, k])
                e[0] = max(float(e[0]), was)
                lo = int(slot[0]) // BLOCK * BLOCK
                to[page[0], lo:int(slot[0])] = _round_e4m3(to[page[0], lo:int(slot[0])] * 2.0 ** (was - float(e[0])))
            to[page, slot] = _round_e4m3(rows[:, a:z] * torch.exp2(-e[nth])[:, None])
    return {"pages": torch.cat([c.reshape(-1, PAGE * LORA), r.reshape(-1, PAGE * ROPE)], 1), "scales": None}
