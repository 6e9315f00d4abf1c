// Prefill hand-off: rows of a prefill into the paged latent cache.
//
// The reference hands prefill states to decode as one flat cache per layer,
// [max_pos][576] bf16 rows c (after kv_a_layernorm) | k_pe (after RoPE), built
// from the hooked kv_a_proj_with_mqa output (src/host/kv_convert.py:36-139)
// and uploaded by the launcher as-is (src/host/fleet_launch.hip:651-669). Here
// the cache is paged, so the hand-off scatters each request's rows into its
// pages: MLA_ROWS_FINAL copies finished rows (the reference's file format);
// MLA_ROWS_RAW takes raw kv_a rows and applies kv_a_layernorm and RoPE at each
// row's position with the same arithmetic as the decode step's appended row.
//
// One warp per row, 8 rows per CTA, grid-stride. Bounds are checked per row:
// a position outside the block table (or, for raw rows, outside the RoPE
// tables) records MLA_DEV_BAD_POSITION and a page id outside the pool records
// MLA_DEV_BAD_PAGE; such rows are skipped. HBM-bound: 1,152 B read and 1,152 B
// written per row.
#include "mla_common.cuh"
#include "mla_kv8.cuh"
#include "mla_rowops.cuh"

namespace mla {

constexpr int kRowsThreads = 256;
constexpr int kRowsPerCta = kRowsThreads / 32;

__global__ void __launch_bounds__(kRowsThreads) k_rows_to_pages(const MlaRowsToPages r) {
    const int lane = threadIdx.x & 31;
    const __nv_bfloat16* rows = reinterpret_cast<const __nv_bfloat16*>(r.rows);
    __nv_bfloat16* cache = reinterpret_cast<__nv_bfloat16*>(r.kv_cache);
    const int64_t n = min(r.total_rows, r.row_start[r.batch]);  // rows past the last request's are nobody's
    for (int64_t i = (int64_t)blockIdx.x * kRowsPerCta + (threadIdx.x >> 5); i < n;
         i += (int64_t)gridDim.x * kRowsPerCta) {
        // request of row i: largest b with row_start[b] <= i
        int lo = 0, hi = r.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (r.row_start[mid] <= i) lo = mid; else hi = mid;
        }
        const int b = lo;
        const int64_t pos64 = (r.first_pos ? r.first_pos[b] : 0) + (i - r.row_start[b]);
        const bool raw = r.mode == MLA_ROWS_RAW;
        if (pos64 < 0 || pos64 >= (int64_t)r.max_blocks * kPage || (raw && pos64 >= r.max_pos)) {
            if (lane == 0) record_error(ErrSink{r.error_word, nullptr}, MLA_DEV_BAD_POSITION);
            continue;
        }
        const int pos = (int)pos64;
        const int page = r.block_table[(int64_t)b * r.max_blocks + pos / kPage];
        if (page < 0 || page >= r.n_pages) {
            if (lane == 0) record_error(ErrSink{r.error_word, nullptr}, MLA_DEV_BAD_PAGE);
            continue;
        }
        const __nv_bfloat16* src = rows + i * r.rows_stride;
        __nv_bfloat16* dst = cache + ((int64_t)page * kPage + pos % kPage) * kRow;
        if (raw) {
            __align__(16) __nv_bfloat16 outc[16];
            float rlo, rhi;
            kv_post_compute(src, reinterpret_cast<const __nv_bfloat16*>(r.kv_a_norm_w), r.rms_eps,
                            r.rope_cos + (int64_t)pos * kRope, r.rope_sin + (int64_t)pos * kRope, lane, outc, rlo,
                            rhi);
            kv_post_store(dst, outc, rlo, rhi, lane);
        } else {
            const uint4* s4 = reinterpret_cast<const uint4*>(src);
            uint4* d4 = reinterpret_cast<uint4*>(dst);
            const uint4 a = s4[lane], c = s4[lane + 32];
            uint4 e = make_uint4(0u, 0u, 0u, 0u);
            if (lane < kRow / 8 - 64) e = s4[lane + 64];
            d4[lane] = a;
            d4[lane + 32] = c;
            if (lane < kRow / 8 - 64) d4[lane + 64] = e;
        }
    }
}

// The same into an 8-bit cache: one CTA per 16-row block that receives rows, two rows
// per warp held in registers, so that every row is read once; the block's largest
// magnitudes meet in shared memory, then the rows are rounded and stored. A first block
// that holds earlier rows of the request keeps the larger of the old and new scales and
// holds those rows anew. 1,152 B read and 576 B written per row: 41 us for 131,072 rows,
// 5.5 TB/s of the copy's 6.45. What keeps it from more is instruction issue (ncu: 238 warp
// instructions per row, the SMs 69 % busy), so values stay packed bf16 pairs until the conversion and
// indexes are 32-bit (before: 280, 76 %, 46 us). Loading the next block ahead in persistent CTAs (64 us), or two blocks per CTA
// (51 us), was slower.
//
// Which block: request b owns the slots row_start[b] / 16 + 2 b .. row_start[b + 1] / 16
// + 2 b + 1, at least as many as the blocks its rows can touch, whatever first_pos is
// (n rows touch at most (n - 1) / 16 + 2 blocks, and floor(x + n) - floor(x) >= floor(n));
// so the grid follows from the totals the host knows, and a slot past a request's last
// block is idle.
__device__ __forceinline__ int64_t block_slot(const MlaRowsToPages& r, int b) {
    return r.row_start[b] / kBlock8 + 2 * (int64_t)b;
}

template <bool raw>
__global__ void __launch_bounds__(kRowsThreads, raw ? 3 : 5) k_rows_to_pages8(const MlaRowsToPages r) {
    static_assert(kRowsPerCta * 2 == kBlock8, "two rows per warp");
    __shared__ alignas(16) float2 red[kRowsPerCta];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t v = blockIdx.x;
    pdl_wait();
    // the request of this slot: largest b with block_slot(b) <= v, 32 probes per round
    int lo = 0, hi = r.batch;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t below = __ballot_sync(0xffffffffu, lane == 0 || (at < hi && block_slot(r, at) <= v));
        lo += (31 - __clz(below)) * step;
        hi = min(hi, lo + step);
    }
    const int b = lo;
    const int64_t row0 = r.row_start[b], n = r.row_start[b + 1] - row0;
    const int64_t first = r.first_pos ? r.first_pos[b] : 0;
    const int64_t nth = v - block_slot(r, b), blk = (first >> 4) + nth;  // 16-row block of the request, rounded down
    static_assert(kBlock8 == 16, "shift by 4");
    if (n <= 0 || nth < 0 || blk > ((first + n - 1) >> 4)) return;
    // rows [p0, p1) of this block
    const int64_t limit = min((int64_t)r.max_blocks * kPage, raw ? (int64_t)r.max_pos : INT64_MAX);
    const int64_t p0 = max(first, blk * kBlock8), p1 = min(first + n, (blk + 1) * kBlock8);
    const ErrSink err{r.error_word, nullptr};
    if ((p0 < 0 || p1 > limit) && threadIdx.x == 0) record_error(err, MLA_DEV_BAD_POSITION);
    if (p0 < 0 || p0 >= limit) return;  // a block is all before position 0 or not at all
    // its rows as slots [a, z) of the block, within the rows given (whatever row_start holds)
    const int64_t base = blk * kBlock8, row_base = row0 - first + base;  // row of the block's slot 0, as it were
    const int a = (int)(p0 - base);
    const int z = (int)max(min(min(p1, limit) - base, r.total_rows - row_base), (int64_t)a);
    if (row_base + a < 0 || z == a) return;
    const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(r.rows) + (row_base + 2 * warp) * r.rows_stride;
    // the rows first, so that the block-table entry's latency overlaps theirs
    RowShare x[2];
    bool has[2], inf = false;
#pragma unroll
    for (int k = 0; k < 2; ++k, src += r.rows_stride) {
        has[k] = 2 * warp + k >= a && 2 * warp + k < z;
        if (!has[k]) continue;
        if (raw) {
            const int64_t pos = base + 2 * warp + k;
            __align__(16) __nv_bfloat16 c[16];
            float lo_f, hi_f;
            kv_post_compute(src, reinterpret_cast<const __nv_bfloat16*>(r.kv_a_norm_w), r.rms_eps,
                            r.rope_cos + pos * kRope, r.rope_sin + pos * kRope, lane, c, lo_f, hi_f);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[k].c[j] = __nv_bfloat162(c[2 * j], c[2 * j + 1]);
            x[k].lo = __float2bfloat16_rn(lo_f);
            x[k].hi = __float2bfloat16_rn(hi_f);
        } else {
            uint4* c = reinterpret_cast<uint4*>(x[k].c);
            c[0] = __ldcs(reinterpret_cast<const uint4*>(src) + 2 * lane);
            c[1] = __ldcs(reinterpret_cast<const uint4*>(src) + 2 * lane + 1);
            x[k].lo = src[kLora + lane];
            x[k].hi = src[kLora + 32 + lane];
        }
    }
    const int page = r.block_table[(int64_t)b * r.max_blocks + p0 / kPage];
    if (page < 0 || page >= r.n_pages) {
        if (threadIdx.x == 0) record_error(err, MLA_DEV_BAD_PAGE);
        return;
    }
    const int slot0 = (int)(base % kPage);
    uint8_t* pg = reinterpret_cast<uint8_t*>(r.kv_cache) + (int64_t)page * kPage8;
    char2* exps = reinterpret_cast<char2*>(r.kv_scales) + (int64_t)page * kBlocks8 + slot0 / kBlock8;
    float ac = 0.f, ar = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (has[k]) inf |= share_amax(x[k], ac, ar);
    // a: earlier rows of the request in this block, which keep their scale at least
    const char2 old = a ? *exps : make_char2(MLA_SCALE_MIN_EXP, MLA_SCALE_MIN_EXP);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        ac = fmaxf(ac, __shfl_xor_sync(0xffffffffu, ac, o));
        ar = fmaxf(ar, __shfl_xor_sync(0xffffffffu, ar, o));
    }
    if (lane == 0) red[warp] = make_float2(ac, ar);
    __syncthreads();  // also: every thread has the old exponents
#pragma unroll
    for (int w = 0; w < kRowsPerCta; w += 2) {
        const float4 m = *reinterpret_cast<const float4*>(&red[w]);
        ac = fmaxf(ac, fmaxf(m.x, m.z));
        ar = fmaxf(ar, fmaxf(m.y, m.w));
    }
    const int e_c = max(scale_exponent(ac), (int)old.x), e_r = max(scale_exponent(ar), (int)old.y);
    if (a) rescale_rows(pg, slot0 / kBlock8, a, pow2i((int)old.x - e_c), pow2i((int)old.y - e_r), threadIdx.x, kRowsThreads);
    if (threadIdx.x == 0) *exps = make_char2((signed char)e_c, (signed char)e_r);
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (has[k]) store_share(pg, slot0 + 2 * warp + k, x[k], inf, e_c, e_r, lane);
}

cudaError_t launch_rows_to_pages(const MlaRowsToPages& r, int sm_count, cudaStream_t stream) {
    if (r.kv_scales) {
        const int64_t slots = r.total_rows / kBlock8 + 2 * (int64_t)r.batch;
        if (r.total_rows <= 0) return cudaSuccess;
        if (slots > INT32_MAX) return cudaErrorInvalidValue;
        if (r.mode == MLA_ROWS_RAW)
            return launch_pdl(k_rows_to_pages8<true>, dim3((unsigned)slots), dim3(kRowsThreads), 0, stream, r);
        return launch_pdl(k_rows_to_pages8<false>, dim3((unsigned)slots), dim3(kRowsThreads), 0, stream, r);
    }
    const int64_t need = (r.total_rows + kRowsPerCta - 1) / kRowsPerCta;
    const int64_t cap = (int64_t)sm_count * 16;
    const int grid = (int)(need < cap ? need : cap);
    if (grid <= 0) return cudaSuccess;
    k_rows_to_pages<<<grid, kRowsThreads, 0, stream>>>(r);
    return cudaGetLastError();
}

}  // namespace mla
