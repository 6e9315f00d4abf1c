// K2 over an 8-bit latent cache — split-KV absorbed-MLA attention on tcgen05.mma
// kind::f8f6f4, with the scores and the output in tensor memory.
//
// Per request, with e4m3 rows C_t (latent c_t, rotary k_t) under the block scales
// 2^ec_t, 2^er_t:
//   s_t[h] = softmax_scale (2^ec_t q_c[h] . c_t + 2^er_t q_pe[h] . k_t)
//   o[h]   = sum_t softmax(s)_t 2^ec_t c_t
//
// Why tensor memory here and m16n8k16 on the bf16 cache: with half the bytes per row
// the SM has half the time per row (25 clocks at the copy peak), and m16n8k16 would
// spend 70 % of its issue on it before a single conversion. An f8f6f4 MMA of K = 32 bytes and
// N = 32 takes 40 clocks at M = 128 and 26 at M = 64 (measured: its shared-memory reads at 128 B
// per clock; 48 at N = 64 by that count), so 128 tokens x 16 heads cost 36 + 16 MMAs, 1,700 of the
// about 3,300 clocks of their HBM time. N is nearly free, so it carries precision: an operand
// that is not 8 bits already enters as a pair of e4m3 values side by side on N,
// x = hi + lo / 16, about as precise as bf16 (8 significant bits) for x in [2^-6, 448]:
//   scores  S^T[t][hi 16 | lo 16] = C[t][:] . Q[hi | lo]   (latent and rotary apart: their scales differ)
//   output  O^T[l][n]            += C^T[l][t] P^T[t][n],  n = hi 16 | lo 16 of P', then of 2^14 P'
// The same tile bytes are the K-major A operand of the scores and the MN-major A
// operand of the output.
//
// The scale of a row enters its probability: P'_t = 2^(s_t + ec_t - m) with m a
// running reference for the largest s_t + ec_t, and the row sum takes
// P'_t 2^-ec_t. P' lies in [0, 256]; a typical largest one is 16, so that a
// later score may exceed the reference 16-fold before the output is rescaled (the
// rescale reads and writes O in tensor memory, which happens in the first few tiles
// of a segment only). A pair of P' alone would end at 2^-14: many rows behind a dominant one,
// as behind an attention sink, would leave the output and still count in the row sum. So a
// P' below 2^-6 is held as the pair of 2^14 P' instead, in 32 columns of its own: 8
// significant bits down to P' = 2^-20, 2^-24 of a typical largest one, fewer below, none
// below 2^-28. The wider N costs an output MMA 8 clocks on 40, and shared memory and tensor
// memory have room for one P and one output instead of two of each (256 x 4096: K2 106.3 us, 104.2
// without). Sums, scores and the output are fp32.
//
// Pages (the plan's units) are TMA'd into a ring of five; a tile is up to two pages of a request. The
// scores are M = 64 MMAs per page, so that a page needs no neighbour in the ring and its scores start
// when it lands. Rows that the query does not see have P' = 0 and, if they share a 32-row step with
// visible ones, are zeroed in the ring (0 times stale NaN bytes would be NaN).
//
// Warps (512 threads):
//   0      TMA producer: pages and their exponents
//   1      score MMAs, owns the tensor memory
//   2      output MMAs
//   3      loads the query of the next segment: K1 left it as the operand's image
//   4-11   softmax: one token and eight heads per thread
//   12-15  partials of a finished segment, while the next one's first scores run (written by the
//          softmax warps, a boundary cost about 2.3 us)
// The MMA warps run their loops as whole warps and elect a lane for the MMAs, so that
// descriptors stay in uniform registers: issued from a lane-0 branch, an MMA took 60-70
// clocks of moving them there.
// Every wait is bounded: a stall records MLA_DEV_TIMEOUT, the roles fall through
// their remaining waits, copies and MMAs drain and the tensor memory is freed.
#include <cuda.h>

#include "mla_kv8.cuh"
#include "mla_tiles.cuh"

namespace mla {

namespace kv8 {

constexpr int kThreads = 512;
constexpr int kSmWarps = 8;                     // softmax warps: 4 token quarters x 2 halves of the heads
constexpr int kSmThreads = kSmWarps * 32;
constexpr int kHh = kHeads / 2;                 // heads of a softmax thread
constexpr int kSlots = 5;                       // ring of pages
constexpr int kEarly = 2;                       // pages requested before the wait on K1
constexpr int kTok = 2 * kPage;                 // tokens per tile
constexpr int kGroup = 8 * kLora;               // 4096: 8 rows of the latent part, [4 column blocks][8][128 B]
constexpr int kSlotC = kPage * kLora;           // 32,768
constexpr int kSlotR = kPage * kRope;           // 4,096
constexpr int kN = kQ8N;                        // hi | lo
constexpr int kNP = 2 * kN;                     // of P', then of 2^14 P'
constexpr int kQ = kQ8C + kQ8R;                 // a request's query image
constexpr int kP = kTok * kNP;                  // [128 tokens][64 B]
constexpr float kPSmall = 0x1p-6f, kPShift = 0x1p14f;  // P' below the first is held as kPShift P'

constexpr int kOffC = 0;
constexpr int kOffR = kOffC + kSlots * kSlotC;
constexpr int kOffQ = kOffR + kSlots * kSlotR;
constexpr int kOffP = kOffQ + 2 * kQ;
constexpr int kOffMisc = kOffP + kP;

struct Smem {
    uint64_t full[kSlots], empty[kSlots];
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2], p_full[2], pv_done[2];
    uint64_t o_full[2], o_empty[2];  // a segment's output complete / written out
    uint64_t ml_full[2];             // its references and row sums
    uint64_t teardown[2];
    uint64_t exps[kSlots];  // a page's 4 x 2 exponents
    alignas(16) float q_scale[2][kQScale];  // [buffer]: per head, then the rotary part's
    alignas(16) float red[2][4][16];
    float m_fin[2][16], lred[2][4][16];  // [segment & 1]
    int32_t pre_cum[65];
    uint32_t tmem_base;
    int abort;
};
constexpr int kSmemBytes = kOffMisc + (int)sizeof(Smem) + 1024;  // + alignment slack
static_assert(kSmemBytes <= 232448, "K2 (8-bit) shared memory exceeds 227 KB");
static_assert(kOffP % 1024 == 0 && kOffQ % 1024 == 0 && kQ % 1024 == 0, "operands must stay 1024-byte aligned");

// Tensor memory columns: two score buffers (per page of the tile: latent 32 | rotary 32), an output of four
// blocks of 64. The scores of a page (M = 64) lie in lanes 0-15 of each warp's 32.
constexpr int kTmemS = 0, kTmemSPage = 2 * kN, kTmemSSize = 2 * kTmemSPage;
constexpr int kTmemO = 2 * kTmemSSize, kTmemCols = 512;
static_assert(kTmemO + 4 * kNP == kTmemCols, "the tensor memory is full");

// Instruction descriptor of kind::f8f6f4 with e4m3 A/B and fp32 D (the fields of
// idesc_bf16_f32; format 0 = e4m3).
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N, int a_mn_major, int b_mn_major) {
    return (1u << 4) | (uint32_t(a_mn_major) << 15) | (uint32_t(b_mn_major) << 16) | (uint32_t(N >> 3) << 17) |
           (uint32_t(M >> 4) << 24);
}
constexpr uint32_t kIdescQK = idesc_e4m3(64, kN, 0, 0);
constexpr uint32_t kIdescPV = idesc_e4m3(128, kNP, 1, 1);

__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Shared-memory descriptor as smem_desc_sw128, with the layout (swizzle) given: 2 =
// 128-byte, 4 = 64-byte; sbo: bytes between groups of 8 rows (K-major)
// or of 8 k (MN-major).
constexpr int kSw128 = 2, kSw64 = 4;
__device__ __forceinline__ uint64_t desc_of(uint32_t saddr, uint32_t sbo_bytes, int layout) {
    return uint64_t((saddr >> 4) & 0x3FFF) | (uint64_t(1) << 16) | (uint64_t((sbo_bytes >> 4) & 0x3FFF) << 32) |
           (uint64_t(1) << 46) | (uint64_t(layout) << 61);
}

__device__ __forceinline__ void tma_load_5d(void* smem_dst, const void* tmap, uint64_t* bar, int x, int y, int z,
                                            int w, int v, uint64_t cache_hint) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v),
        "l"(cache_hint)
        : "memory");
}

// A CTA's tiles: one or two plan units (pages) of one request.
struct Walk : TileCursor {
    __device__ int pages() const { return u + 1 < u_end && u + 1 < cb1 ? 2 : 1; }
    __device__ bool last() const { return u + pages() == u_end || u + pages() == cb1; }
    __device__ void next() {
        u += pages() - 1;
        TileCursor::next();
    }
    __device__ void next_request() {
        u = min(cb1, u_end) - 1;
        TileCursor::next();
    }
};

// Whether any row of the tile's 32-row step ks is visible.
__device__ __forceinline__ bool step_on(const Visible& v, int index, int pages, int ks) {
    if ((ks >> 1) >= pages) return false;
    const int r0 = kPage * v.tile(index + (ks >> 1)) + 32 * (ks & 1);
    return r0 < v.rows && (r0 < v.head || r0 + 32 > v.lo);
}

// The rest of a bounded wait whose first try failed; once a role gave up, every other wait falls
// through at once. Out of line: the waits are many, and a CTA's first tile runs from a cold
// instruction cache.
__device__ __noinline__ bool slow_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int32_t* error_word,
                                       int32_t* error_host) {
    if (*abort) return false;
    return mbar_wait(bar, parity, abort, ErrSink{error_word, error_host});
}

__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(r));
    return r != 0;
}

// 8 consecutive tensor-memory columns of 32 lanes (tmem_ld16, half as wide), and back.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[kHh]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(taddr));
}
// 8 score columns of a warp's 16 rows of either page: threads 0-15 the first page's, 16-31 the second's.
__device__ __forceinline__ void tmem_ld8_pages(uint32_t taddr, float (&v)[kHh]) {
    asm volatile("tcgen05.ld.sync.aligned.16x32bx2.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8], %9;"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(taddr), "n"(kTmemSPage));
}
// The loaded values, not to be used before the tmem_wait_ld that precedes this call.
__device__ __forceinline__ void loaded(float (&v)[kHh]) {
    asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float (&v)[kHh]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                 "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}

// An untiled copy global -> shared, completing on an mbarrier (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(smem_dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// Reduction of 8 values over the 32 lanes of a warp by halving exchanges: lanes 4 h ..
// 4 h + 3 end with value h.
template <bool kMax>
__device__ __forceinline__ float reduce8(const float (&v)[kHh], int lane) {
    auto op = [](float a, float b) { return kMax ? fmaxf(a, b) : a + b; };
    float r4[4], r2[2];
    const bool b4 = lane & 16, b3 = lane & 8, b2 = lane & 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float send = b4 ? v[j] : v[j + 4], keep = b4 ? v[j + 4] : v[j];
        r4[j] = op(keep, __shfl_xor_sync(0xffffffffu, send, 16));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float send = b3 ? r4[j] : r4[j + 2], keep = b3 ? r4[j + 2] : r4[j];
        r2[j] = op(keep, __shfl_xor_sync(0xffffffffu, send, 8));
    }
    const float send = b2 ? r2[0] : r2[1], keep = b2 ? r2[1] : r2[0];
    float r = op(keep, __shfl_xor_sync(0xffffffffu, send, 4));
    r = op(r, __shfl_xor_sync(0xffffffffu, r, 2));
    return op(r, __shfl_xor_sync(0xffffffffu, r, 1));
}

}  // namespace kv8

__global__ void __launch_bounds__(kv8::kThreads, 1)
    k2_attention_kv8(const MlaDecodeParams p, const __grid_constant__ CUtensorMap tmap_c,
                     const __grid_constant__ CUtensorMap tmap_r, float scale_log2) {
    using namespace kv8;
    MLA_TL_SCOPE(1);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Smem& S = *reinterpret_cast<Smem*>(smem + kOffMisc);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    const WsLayout ws = ws_layout(p);
    char* wsb = reinterpret_cast<char*>(p.workspace);
    const ErrSink err = err_sink(p);
    const int fresh = new_row_count(p);

    pdl_trigger();
    const int vc = blockIdx.x;

    // Set-up, side by side: warp 1 takes the tensor memory, warp 2 makes the barriers, and warp 0
    // the split plan: for up to 64 requests from the step's inputs, before the wait on K1 (the rule
    // K1's planner uses); beyond, all read K1's plan entry after it.
    constexpr int kPrePlan = 64;
    int32_t* pre_cum = S.pre_cum;
    const bool pre = p.batch <= kPrePlan;
    if (warp == 0) {
        if (pre) {
            const int b0 = 2 * lane, b1 = b0 + 1;
            const int n0 = b0 < p.batch ? plan_tiles(p, b0) : 0, n1 = b1 < p.batch ? plan_tiles(p, b1) : 0;
            int incl = n0 + n1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            pre_cum[b0] = incl - n0 - n1;  // beyond the batch: the total
            pre_cum[b1] = incl - n1;
            if (lane == 31) pre_cum[kPrePlan] = incl;
        }
    } else if (warp == 1) {
        tmem_alloc(&S.tmem_base, kTmemCols);
        tmem_relinquish();
    } else if (warp == 2 && lane == 0) {
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&S.full[i], 2);  // the copies, the exponents
            mbar_init(&S.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&S.q_full[i], 1);
            mbar_init(&S.q_empty[i], 1 + kSmWarps);
            mbar_init(&S.s_full[i], 1);
            mbar_init(&S.p_full[i], kSmWarps);
            mbar_init(&S.pv_done[i], 1);
            mbar_init(&S.teardown[i], 1);
            mbar_init(&S.o_full[i], 1);
            mbar_init(&S.o_empty[i], 4);
            mbar_init(&S.ml_full[i], kSmWarps);
        }
        S.abort = 0;
        fence_mbar_init();
    } else if (warp == 3 && lane == 0) {
        prefetch_tmap(&tmap_c);
        prefetch_tmap(&tmap_r);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    const int32_t* cum = reinterpret_cast<const int32_t*>(wsb + ws.tiles_cum);
    PlanEntry pe{};
    int G;
    if (pre) {
        cum = pre_cum;
        const int64_t U = pre_cum[p.batch];
        G = (int)(U < (int64_t)p.num_ctas ? U : (int64_t)p.num_ctas);
        if (vc < G) {
            pe.u_begin = plan_begin(vc, U, G);
            pe.u_end = plan_begin(vc + 1, U, G);
            int lo = 0, hi = p.batch;  // largest b with cum[b] <= u_begin (skips empty requests)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (pre_cum[mid] <= pe.u_begin) lo = mid; else hi = mid;
            }
            pe.b = lo;
            pe.cb0 = pre_cum[lo];
            pe.cb1 = pre_cum[lo + 1];
        }
    } else {
        pdl_wait();
        MLA_TL_WAITED(1);
        G = reinterpret_cast<const PlanHeader*>(wsb + ws.plan)->G;
        pe = reinterpret_cast<const PlanEntry*>(wsb + ws.plan + sizeof(PlanHeader))[vc < p.num_ctas ? vc : 0];
    }
    const uint32_t tmem = __shfl_sync(0xffffffffu, S.tmem_base, 0);
    if (vc >= G) {  // uniform per CTA: no work
        if (pre) pdl_wait();
        if (warp == 1) tmem_dealloc(tmem, kTmemCols);
        return;
    }
    volatile int* abort = &S.abort;
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        return mbar_try_wait(bar, parity) || slow_wait(bar, parity, abort, p.error_word, p.error_host);
    };

    Walk cur;
    cur.init_at(cum, p.seq_lens, p.batch, pe, fresh);
    auto visible = [&](int b) { return Visible(p, p.seq_lens[b] + fresh, kPage); };

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        // A page's number is loaded two pages ahead and its exponents one page ahead, so that neither
        // latency is on the path; they join the page's barrier after its copies were issued. Up to
        // kEarly pages go out before the wait on K1, none that K1 appends to (and whose exponents it
        // may raise).
        if (lane == 0) {
            struct Page { int id; bool appended; };
            TileCursor la = cur;  // two pages ahead of the one being loaded
            Visible vis;
            auto page_of = [&]() -> Page {
                if (la.first()) vis = visible(la.b);
                const int k = vis.tile(la.index());
                return Page{p.block_table[(int64_t)la.b * p.max_blocks + k], fresh && k == (vis.rows - 1) / kPage};
            };
            auto page_ok = [&](int id) { return id >= 0 && id < p.n_pages; };
            auto exps_of = [&](int id) { return reinterpret_cast<const uint64_t*>(p.kv_scales)[page_ok(id) ? id : 0]; };
            bool waited = !pre;
            Page p0 = page_of(), p1 = p0, p2 = p0;
            la.next();
            if (la.valid()) p1 = page_of();
            uint64_t ex0 = 0, ex1 = 0;
            bool early0 = true, early1 = true;  // not loaded yet, or before the wait
            uint32_t i = 0;
            TileCursor at = cur;
            for (; at.valid(); at.next(), ++i) {
                if (!waited && (i >= kEarly || p0.appended)) { pdl_wait(); MLA_TL_WAITED(1); waited = true; }
                const uint32_t sl = i % kSlots;
                if (i >= kSlots && !wait(&S.empty[sl], (i / kSlots - 1) & 1)) break;
                if (!page_ok(p0.id)) record_error(err, MLA_DEV_BAD_PAGE);
                const int id = page_ok(p0.id) ? p0.id : 0;
                mbar_arrive_expect_tx(&S.full[sl], kSlotC + kSlotR);
                tma_load_5d(smem + kOffC + sl * kSlotC, &tmap_c, &S.full[sl], 0, 0, 0, 0, id, kCacheEvictFirst);
                tma_load_3d(smem + kOffR + sl * kSlotR, &tmap_r, &S.full[sl], 0, 0, id, kCacheEvictFirst);
                if (i == 0 || (p0.appended && early0)) ex0 = exps_of(id);
                la.next();
                if (la.valid()) p2 = page_of();
                ex1 = exps_of(p1.id);
                early1 = !waited;
                S.exps[sl] = ex0;
                mbar_arrive(&S.full[sl]);
                p0 = p1; p1 = p2; ex0 = ex1; early0 = early1;
            }
            if (!waited) pdl_wait();
            // Drain: every issued copy must land before the CTA's shared memory is released.
            for (uint32_t sl = 0; sl < kSlots; ++sl) {
                const uint32_t fills = i / kSlots + (sl < i % kSlots ? 1u : 0u);
                if (fills) mbar_drain(&S.full[sl], (fills - 1) & 1, err);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ score MMAs
        const uint64_t dc = desc_of(smem_u32(smem + kOffC), kGroup, kSw128);
        const uint64_t dr = desc_of(smem_u32(smem + kOffR), 8 * kRope, kSw64);
        const uint64_t dqc = desc_of(smem_u32(smem + kOffQ), 1024, kSw128);
        const uint64_t dqr = desc_of(smem_u32(smem + kOffQ + kQ8C), 8 * kRope, kSw64);
        uint32_t j = 0, i = 0;  // tile, page
        bool ok = true;
        for (; ok && cur.valid(); cur.next(), ++j) {
            const uint32_t qb = cur.seg & 1, sb = j & 1;
            const int pages = cur.pages();
            const bool last = cur.last();
            ok = !cur.first() || wait(&S.q_full[qb], (cur.seg >> 1) & 1);
            ok &= j < 2 || wait(&S.p_full[sb], ((j - 2) >> 1) & 1);  // the buffer's scores were read
            const uint64_t b = dqc + ((qb * kQ) >> 4), br = dqr + ((qb * kQ) >> 4);
            for (int k = 0; k < pages; ++k, ++i) {
                const uint32_t sl = i % kSlots;
                ok &= wait(&S.full[sl], (i / kSlots) & 1);
                ok = __all_sync(0xffffffffu, ok);  // one answer for the warp, even if a wait ran out in some lanes
                if (!ok) break;
                tc_fence_after();
                const uint64_t a = dc + ((sl * kSlotC) >> 4), ar = dr + ((sl * kSlotR) >> 4);
                const uint32_t d = tmem + kTmemS + kTmemSSize * sb + kTmemSPage * k;
                if (elect_one()) {
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        mma_f8(d, a + (((x >> 2) * 1024 + (x & 3) * 32) >> 4),
                               b + (((x >> 2) * (kN * 128) + (x & 3) * 32) >> 4), kIdescQK, x > 0);
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        mma_f8(d + kN, ar + ((x * 32) >> 4), br + ((x * 32) >> 4), kIdescQK, x > 0);
                    if (k == pages - 1) {
                        tc_commit(&S.s_full[sb]);
                        if (last) tc_commit(&S.q_empty[qb]);
                    }
                }
                __syncwarp();
            }
        }
        __syncwarp();
        if (elect_one()) {  // all issued MMAs complete before the tensor memory is freed
            tc_commit(&S.teardown[0]);
            mbar_drain(&S.teardown[0], 0, err);
        }
    } else if (warp == 2) {
        // ------------------------------------------------------------ output MMAs
        const uint64_t dc = desc_of(smem_u32(smem + kOffC), kGroup, kSw128);
        const uint64_t dp = desc_of(smem_u32(smem + kOffP), 8 * kNP, kSw64);
        Visible vis;
        uint32_t j = 0, i = 0;
        for (; cur.valid(); i += cur.pages(), cur.next(), ++j) {
            const uint32_t sb = j & 1, ob = cur.seg & 1;
            const bool first = cur.first(), last = cur.last();
            const int pages = cur.pages();
            if (first) vis = visible(cur.b);
            uint32_t on = 0;  // bit ks: the 32-row step ks holds a visible row
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) on |= (uint32_t)step_on(vis, cur.index(), pages, ks) << ks;
            const uint32_t sl0 = i % kSlots, sl1 = (i + 1) % kSlots;
            bool ok = wait(&S.p_full[sb], (j >> 1) & 1);
            ok &= !first || cur.seg < 1 || wait(&S.o_empty[ob ^ 1], ((cur.seg - 1) >> 1) & 1);
            ok &= wait(&S.full[sl0], (i / kSlots) & 1);
            ok &= pages < 2 || wait(&S.full[sl1], ((i + 1) / kSlots) & 1);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            const uint64_t a0 = dc + ((sl0 * kSlotC) >> 4), a1 = dc + ((sl1 * kSlotC) >> 4);
            const uint32_t d = tmem + kTmemO;
            if (elect_one()) {
                uint32_t acc = first ? 0u : 1u;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    if ((on >> ks) & 1) {
                        const uint64_t a = (ks < 2 ? a0 : a1) + (((ks & 1) * 4 * kGroup) >> 4);
#pragma unroll
                        for (int cb = 0; cb < 4; ++cb)
                            mma_f8(d + kNP * cb, a + ((cb * 1024) >> 4), dp + ((ks * 32 * kNP) >> 4), kIdescPV, acc);
                        acc = 1u;
                    }
                    if (ks == 1) tc_commit(&S.empty[sl0]);
                    if (ks == 3 && pages > 1) tc_commit(&S.empty[sl1]);
                }
                tc_commit(&S.pv_done[sb]);
                if (last) tc_commit(&S.o_full[ob]);
            }
            __syncwarp();
        }
        __syncwarp();
        if (elect_one()) {
            tc_commit(&S.teardown[1]);
            mbar_drain(&S.teardown[1], 0, err);
        }
    } else if (warp == 3) {
        // ------------------------------------------------------------ queries
        if (lane == 0) {
            if (pre) pdl_wait();
            const char* img = wsb + ws.qa;
            const float* q_scale = reinterpret_cast<const float*>(wsb + ws.q_scale);
            uint32_t issued = 0;
            for (; cur.valid(); cur.next_request(), ++issued) {
                const uint32_t qb = cur.seg & 1;
                if (cur.seg >= 2 && !wait(&S.q_empty[qb], ((cur.seg >> 1) - 1) & 1)) break;
                mbar_arrive_expect_tx(&S.q_full[qb], kQ + kQScale * 4);
                bulk_load(smem + kOffQ + qb * kQ, img + (int64_t)cur.b * kQ, kQ, &S.q_full[qb]);
                bulk_load(S.q_scale[qb], q_scale + (int64_t)cur.b * kQScale, kQScale * 4, &S.q_full[qb]);
            }
            for (uint32_t qb = 0; qb < 2; ++qb) {  // drained as the pages are
                const uint32_t fills = issued / 2 + (qb < issued % 2 ? 1u : 0u);
                if (fills) mbar_drain(&S.q_full[qb], (fills - 1) & 1, err);
            }
        }
    } else if (warp >= 12) {
        // ------------------------------------------------------------ partials
        // Thread: latent column 32 sp + lane of each 128-column block, all 16 heads.
        const int sp = warp & 3;
        float* part_ml = reinterpret_cast<float*>(wsb + ws.part_ml);
        float* part_acc = reinterpret_cast<float*>(wsb + ws.part_acc);
        if (pre) pdl_wait();  // the previous step's merge has read the partials
        for (; cur.valid(); cur.next_request()) {
            const uint32_t ob = cur.seg & 1, ph = (cur.seg >> 1) & 1;
            const int64_t part = (int64_t)vc + cur.b;
            wait(&S.ml_full[ob], ph);
            if (sp == 0 && lane < kHeads) {
                const float l = (S.lred[ob][0][lane] + S.lred[ob][1][lane]) + (S.lred[ob][2][lane] + S.lred[ob][3][lane]);
                *reinterpret_cast<float2*>(part_ml + (part * kHeads + lane) * 2) = make_float2(S.m_fin[ob][lane], l);
            }
            __syncwarp();
            wait(&S.o_full[ob], ph);
            tc_fence_after();
            __syncwarp();
            float* acc = part_acc + part * kHeads * kLora + 32 * sp + lane;
#pragma unroll 2
            for (int k = 0; k < 8; ++k) {  // four blocks, two halves of the heads
                float o[kHh], q[kHh], so[kHh], sq[kHh];
                const uint32_t ta = tmem_lane_addr(tmem, sp, kTmemO + kNP * (k >> 1) + kHh * (k & 1));
                tmem_ld8(ta, o);
                tmem_ld8(ta + kHeads, q);
                tmem_ld8(ta + kN, so);
                tmem_ld8(ta + kN + kHeads, sq);
                tmem_wait_ld();
                loaded(o); loaded(q); loaded(so); loaded(sq);
#pragma unroll
                for (int h = 0; h < kHh; ++h)
                    acc[(kHh * (k & 1) + h) * kLora + 128 * (k >> 1)] =
                        fmaf(fmaf(sq[h], 0.0625f, so[h]), 1.f / kPShift, fmaf(q[h], 0.0625f, o[h]));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.o_empty[ob]);
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------ softmax
        // Threads 0-15 of a warp hold rows 16 sp .. of the tile's first page, 16-31 those of the second.
        const int sp = warp & 3, half = lane >> 4, slot = 16 * sp + (lane & 15), tok = half * kPage + slot;
        const int h0 = warp < 8 ? 0 : kHh;  // this thread's heads: h0 .. h0 + 7
        float m[kHh], l[kHh];  // reference (log2 domain), this thread's part of the row sum
        float qs[kHh], qsr = 0.f;  // what this thread's heads' scores are multiplied by, latent and rotary
        Visible vis;
        uint32_t j = 0, i0 = 0;  // tile, its first page
        // The first pass is a rehearsal without a visible row, while the first tile is on its way: it
        // fetches the code (measured: 3,000 clocks for a first tile from a cold cache, 1,000 for a later
        // one). It waits for nothing, signals nothing and stores nothing that is not written again.
        for (bool dry = true; dry || cur.valid();) {
            const uint32_t sb = j & 1, sl0 = i0 % kSlots, sl1 = (i0 + 1) % kSlots, sl = half ? sl1 : sl0;
            const bool first = cur.first(), last = cur.last();
            if (first) vis = visible(cur.b);
            const int index = cur.index(), pages = cur.pages();
            const bool sees = !dry && half < pages && vis.row(kPage * vis.tile(index + half) + slot);
            if (!dry) {  // the exponents, and the pages themselves where rows are zeroed
                wait(&S.full[sl0], (i0 / kSlots) & 1);
                if (pages > 1) wait(&S.full[sl1], ((i0 + 1) / kSlots) & 1);
            }
            const char2 ex = sees ? reinterpret_cast<const char2*>(&S.exps[sl])[slot / kBlock8] : make_char2(0, 0);
            if (first) {
                const int qb = cur.seg & 1;
                if (!dry) wait(&S.q_full[qb], (cur.seg >> 1) & 1);
                qsr = S.q_scale[qb][kHeads] * scale_log2;
#pragma unroll
                for (int h = 0; h < kHh; ++h) qs[h] = S.q_scale[qb][h0 + h] * scale_log2;
                __syncwarp();
                if (!dry && lane == 0) mbar_arrive(&S.q_empty[qb]);
#pragma unroll
                for (int h = 0; h < kHh; ++h) { m[h] = -INFINITY; l[h] = 0.f; }
            }
            const float fc = pow2i(ex.x), fr = pow2i(ex.y) * qsr, e = (float)ex.x;
            if (!dry) wait(&S.s_full[sb], (j >> 1) & 1);
            tc_fence_after();
            __syncwarp();
            float s[kHh];
            {
                float a[kHh], b[kHh], c[kHh];
                const uint32_t ta = tmem_lane_addr(tmem, sp, kTmemS + kTmemSSize * sb + h0);
                tmem_ld8_pages(ta, s);
                tmem_ld8_pages(ta + 16, a);
                tmem_ld8_pages(ta + 32, b);
                tmem_ld8_pages(ta + 48, c);
                tmem_wait_ld();
                loaded(s); loaded(a); loaded(b); loaded(c);
#pragma unroll
                for (int h = 0; h < kHh; ++h)
                    s[h] = sees ? fmaf(fmaf(a[h], 0.0625f, s[h]), fc * qs[h], fmaf(fmaf(c[h], 0.0625f, b[h]), fr, e)) : -INFINITY;
            }
            // ---- the reference per head: kept unless a score exceeds it 256-fold (16-fold the
            // largest so far); the first tile of a segment sets it ----
            bool exchange = first;
            if (!first) {
                bool over = false;
#pragma unroll
                for (int h = 0; h < kHh; ++h) over |= s[h] > m[h] + 8.f;
                exchange = bar_red_or(1, kSmThreads, over);
            }
            if (exchange) {
                const float wmax = reduce8<true>(s, lane);
                if ((lane & 3) == 0) S.red[sb][sp][h0 + (lane >> 2)] = wmax;
                named_bar_sync(1, kSmThreads);
                float f[kHh], t[kHh];
#pragma unroll
                for (int k = 0; k < kHh; k += 4) {
                    float4 x = *reinterpret_cast<const float4*>(&S.red[sb][0][h0 + k]);
#pragma unroll
                    for (int w = 1; w < 4; ++w) {
                        const float4 y = *reinterpret_cast<const float4*>(&S.red[sb][w][h0 + k]);
                        x = make_float4(fmaxf(x.x, y.x), fmaxf(x.y, y.y), fmaxf(x.z, y.z), fmaxf(x.w, y.w));
                    }
                    t[k] = x.x; t[k + 1] = x.y; t[k + 2] = x.z; t[k + 3] = x.w;
                }
#pragma unroll
                for (int h = 0; h < kHh; ++h) {
                    const float n = fmaxf(m[h], t[h] - 4.f);
                    f[h] = first ? 1.f : fast_exp2(m[h] - n);
                    m[h] = n;
                    l[h] *= f[h];
                }
                if (!first) {
                    wait(&S.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1);
                    tc_fence_after();
                    __syncwarp();
#pragma unroll 2
                    for (int k = 0; k < 4 * kNP / kHeads; ++k) {  // four blocks of two pairs
                        float o[kHh];
                        const uint32_t ta = tmem_lane_addr(tmem, sp, kTmemO + kHeads * k + h0);
                        tmem_ld8(ta, o);
                        tmem_wait_ld();
                        loaded(o);
#pragma unroll
                        for (int h = 0; h < kHh; ++h) o[h] *= f[h];
                        tmem_st8(ta, o);
                    }
                    tmem_wait_st();
                }
            }
            // ---- P' as e4m3 pairs, the row sums over the unrounded values ----
            const float back = pow2i(-(int)ex.x);
            uint32_t hi[2], lo[2], small[2];  // four heads each; small: 0xFF where the pair is of 2^14 P'
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t x[2], y[2];
                small[k] = 0;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int h = 4 * k + 2 * i;
                    float u = sees ? fast_exp2(s[h] - m[h]) : 0.f, w = sees ? fast_exp2(s[h + 1] - m[h + 1]) : 0.f;
                    l[h] = fmaf(u, back, l[h]);
                    l[h + 1] = fmaf(w, back, l[h + 1]);
                    if (u < kPSmall) { u *= kPShift; small[k] |= 0xFFu << (16 * i); }
                    if (w < kPSmall) { w *= kPShift; small[k] |= 0xFF00u << (16 * i); }
                    e4m3_pairs(u, w, x[i], y[i]);
                }
                hi[k] = x[0] | (x[1] << 16);
                lo[k] = y[0] | (y[1] << 16);
            }
            if (j >= 1) wait(&S.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1);  // the last tile's P was read
            {
                uint8_t* pt = smem + kOffP + tok * kNP + h0;
                const int sw = (tok >> 1) & 3;
                *reinterpret_cast<uint2*>(pt + (sw << 4)) = make_uint2(hi[0] & ~small[0], hi[1] & ~small[1]);
                *reinterpret_cast<uint2*>(pt + ((sw ^ 1) << 4)) = make_uint2(lo[0] & ~small[0], lo[1] & ~small[1]);
                *reinterpret_cast<uint2*>(pt + ((sw ^ 2) << 4)) = make_uint2(hi[0] & small[0], hi[1] & small[1]);
                *reinterpret_cast<uint2*>(pt + ((sw ^ 3) << 4)) = make_uint2(lo[0] & small[0], lo[1] & small[1]);
            }
            if (!sees && !dry && step_on(vis, index, pages, 2 * half + (slot >> 5))) {  // 0 * stale bytes must be 0
                uint8_t* row = smem + kOffC + sl * kSlotC + (slot >> 3) * kGroup + (slot & 7) * 128 + (h0 >> 3) * 2048;
#pragma unroll 4
                for (int i = 0; i < kLora / 32; ++i)  // this half's two column blocks
                    *reinterpret_cast<uint4*>(row + (i >> 3) * 1024 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            tc_fence_before();
            __syncwarp();
            if (!dry && lane == 0) mbar_arrive(&S.p_full[sb]);

            if (last || dry) {  // the segment's references and row sums, for the partial
                const uint32_t ob = cur.seg & 1;
                const float ls = reduce8<false>(l, lane);
                if (cur.seg >= 2) wait(&S.o_empty[ob], ((cur.seg >> 1) - 1) & 1);
                if ((lane & 3) == 0) S.lred[ob][sp][h0 + (lane >> 2)] = ls;
                if (sp == 0 && lane == 0) {
#pragma unroll
                    for (int h = 0; h < kHh; ++h) S.m_fin[ob][h0 + h] = m[h];
                }
                __syncwarp();
                if (!dry && lane == 0) mbar_arrive(&S.ml_full[ob]);
            }
            if (dry) {
                dry = false;
                continue;
            }
            i0 += pages;
            cur.next();
            ++j;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

cudaError_t k2_kv8_configure() {
    return cudaFuncSetAttribute(k2_attention_kv8, cudaFuncAttributeMaxDynamicSharedMemorySize, kv8::kSmemBytes);
}

cudaError_t launch_attention_kv8(const MlaDecodeParams& p, const CUtensorMap& tmap_c, const CUtensorMap& tmap_r,
                                 float scale_log2, cudaStream_t stream) {
    const cudaError_t e = launch_pdl(k2_attention_kv8, dim3(p.num_ctas), dim3(kv8::kThreads), kv8::kSmemBytes, stream,
                                     p, tmap_c, tmap_r, scale_log2);
    if (e != cudaSuccess) return e;
    return cudaGetLastError();
}

}  // namespace mla
