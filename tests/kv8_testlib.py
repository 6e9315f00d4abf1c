"""64-bit restatements of the 8-bit cache and of windowed decode attention, for the tests.

Written from the definitions, in NumPy, apart from the library: an e4m3 value is the nearest
one with ties to even; a block of 16 rows of a part has the exponent
min{e >= -64 : amax <= 448 * 2^e} over the rows it ever held, raised in the order rows join.
"""
import numpy as np

HEADS, NOPE, ROPE, V, LORA, ROW, PAGE, BLOCK = 16, 128, 64, 128, 512, 576, 64, 16
PARTS = ((0, LORA), (LORA, ROW))


def bf16(x):
    """Round to bf16 (nearest, ties to even), as float64. Non-finite values stay."""
    x = np.asarray(x, np.float64)
    m, e = np.frexp(np.where(np.isfinite(x), x, 0.0))
    step = np.exp2(np.maximum(e, -125) - 8.0)
    return np.where(np.isfinite(x), np.rint(np.where(np.isfinite(x), x, 0.0) / step) * step, x)


def round_e4m3(x):
    """Nearest e4m3 value of |x| <= 448; infinities become NaN."""
    ok = np.isfinite(x)
    y = np.where(ok, x, 0.0)
    e = np.maximum(np.frexp(np.abs(y))[1] - 1, -6)
    step = np.exp2(e - 3.0)
    return np.where(ok, np.rint(y / step) * step, np.nan)


def exponent(rows):
    """The exponent of a set of rows (of one part)."""
    a = np.abs(rows[np.isfinite(rows)])
    a = float(a.max()) if a.size else 0.0
    e = -64
    while a > 448.0 * 2.0 ** e:
        e += 1
    return e


class Cache8:
    """One request's rows in an 8-bit cache: codes (e4m3 values) and exponents per block and part."""

    def __init__(self, n_rows):
        n_blocks = -(-n_rows // BLOCK)
        self.codes = np.zeros((n_blocks * BLOCK, ROW))
        self.exps = np.zeros((n_blocks, 2), np.int64)

    def write(self, first, rows):
        """Store rows at positions first .. in one call."""
        for blk in range(first // BLOCK, (first + len(rows) - 1) // BLOCK + 1 if len(rows) else 0):
            p0, p1 = max(first, blk * BLOCK), min(first + len(rows), (blk + 1) * BLOCK)
            new = rows[p0 - first:p1 - first]
            for k, (a, b) in enumerate(PARTS):
                e = exponent(new[:, a:b])
                if p0 > blk * BLOCK:
                    old = self.exps[blk, k]
                    e = max(e, int(old))
                    before = slice(blk * BLOCK, p0)
                    self.codes[before, a:b] = round_e4m3(self.codes[before, a:b] * 2.0 ** (int(old) - e))
                self.exps[blk, k] = e
                self.codes[p0:p1, a:b] = round_e4m3(new[:, a:b] * 2.0 ** -e)

    def values(self, n):
        f = np.exp2(np.repeat(self.exps.astype(np.float64), BLOCK, 0))[:n]
        return self.codes[:n] * np.concatenate([np.repeat(f[:, :1], LORA, 1), np.repeat(f[:, 1:], ROPE, 1)], 1)


def read_request(cache, b, n):
    """(codes [n, 576], exponents [blocks, 2]) of request b's first n rows, from a PagedLatentCache8."""
    table = cache.block_table[b].cpu().numpy()
    pages = cache.pages.view(__import__("torch").float8_e4m3fn).float().cpu().numpy().astype(np.float64)
    scales = cache.scales.cpu().numpy().astype(np.int64)
    got = np.zeros((n, ROW))
    for t in range(n):
        pg, sl = table[t // PAGE], t % PAGE
        got[t, :LORA] = pages[pg, sl * LORA:(sl + 1) * LORA]
        got[t, LORA:] = pages[pg, PAGE * LORA + sl * ROPE:PAGE * LORA + (sl + 1) * ROPE]
    exps = np.stack([scales[table[t // PAGE], t % PAGE // BLOCK] for t in range(0, n, BLOCK)]) if n else np.zeros((0, 2))
    return got, exps


def visible(n, window, sinks):
    """Rows that the query at row n sees."""
    t = np.arange(n + 1)
    return t if not window else t[(t < sinks) | (t > n - window)]


def rope(x, cos, sin):
    """Interleaved pairs rotated; halves of the result (x [..., 64], cos / sin [64])."""
    e, o = x[..., 0::2], x[..., 1::2]
    return np.concatenate([e * cos[:32] - o * sin[:32], o * cos[32:] + e * sin[32:]], -1)


def attention(q, rows, kv_b, cos, sin, scale):
    """(out [2048], bound scale [2048], score change [2048]) of one query [3072] over its visible rows
    [n, 576], in 64 bits; the rotated query is bf16, as the model defines it (reference_decode.py:235).
    The second array is sum_l |W_UV| sum_t p_t |c_t|: what relative errors of p multiply."""
    q = q.reshape(HEADS, NOPE + ROPE)
    w = kv_b.reshape(HEADS, NOPE + V, LORA)
    qa = np.concatenate([np.einsum("hd,hdc->hc", q[:, :NOPE], w[:, :NOPE]), bf16(rope(q[:, NOPE:], cos, sin))], 1)
    s = qa @ rows.T * scale
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    out = np.einsum("hvc,hc->hv", w[:, NOPE:], p @ rows[:, :LORA])
    mag = np.einsum("hvc,hc->hv", np.abs(w[:, NOPE:]), p @ np.abs(rows[:, :LORA]))
    # the largest change of a score when every product is off by 2^-9 (the absorbed query is bf16)
    ds = scale * 2.0 ** -9 * (np.abs(qa) @ np.abs(rows).T).max(1)
    return out.reshape(-1), mag.reshape(-1), np.repeat(ds, V)


def check_out(got, out, mag, ds, what=""):
    """An output against its 64-bit value. Derivation of the bound, per element: the output is rounded
    to bf16 (2^-9 relative); probabilities are off by up to 2^-8 (a pair of e4m3 values, or bf16) and
    by the change of their score, 2 ds with the normalisation; everything else (fp32 sums) is far below.
    Over all elements these errors are independent, so the 2-norm is held to 2^-8 of the output's
    where no element is dominated by cancellation."""
    tol = np.abs(out) * 2.0 ** -8 + mag * (2.0 ** -8 + 2 * ds) + 1e-30
    bad = ~(np.abs(got - out) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} elements off, worst {np.nanmax(np.abs(got - out) / tol):.2f} of the bound"
