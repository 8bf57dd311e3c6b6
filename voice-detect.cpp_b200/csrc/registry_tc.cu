// Many queries against the quantised registry on the tensor cores: their scores, or their
// posterior without storing the scores.
//
//   1. registry_prepare_kernel: each query's unit vector as two f16 parts (hi | lo), and the
//      stored rows as f16 whole numbers (exact), once per call, with a table of each row's
//      factor (temperature log2(e) scale, and -2e30 for an empty slot), so that one fused
//      multiply-add turns an accumulator into a base-2 logit.
//   2. registry_tc_kernel: a persistent tcgen05 product, 128 queries x 256 rows a tile, both
//      parts of the query accumulated into one f32 accumulator in TMEM (two buffers). Its
//      epilogue (thread = query) stores the scores, or sums the softmax of every 8-row chunk
//      and keeps only the best logits of the chunks and of groups of sixteen; the chunk that
//      holds the thread's best score so far stays apart from the sums, so that a sum next to
//      0 is not lost under the top score.
//   3. registry_answer_kernel (posterior): the best L = k + 4 chunks of each query by (best
//      logit, lower chunk) - any score outside them is behind one score of each -, their
//      scores again from the stored codes, the best L of those rescored in f64.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <mutex>

#include "batches.h"
#include "registry.cuh"

namespace vdb {
namespace {

constexpr int kTcThreads = 384;  // warp 0 TMA, warp 1 MMA, warps 4..11 epilogue
constexpr int kTcQ = 128;        // queries per tile (MMA M)
constexpr int kTcRows = 256;     // registry rows per tile (MMA N)
constexpr int kChunk = 8;        // rows per chunk: what step 3 scores again for one hot logit
constexpr int kGroup = 16;       // chunks per group (one thread's columns of a tile)
constexpr int kTabs = 4;         // row tables in flight
constexpr uint32_t kTabBytes = 2 * kTcRows * 4;
constexpr uint32_t kResBytes = kTcQ * 64 * 2;   // resident query box: 64 dims, 128 B rows
constexpr uint32_t kRowBoxBytes = kTcRows * 32 * 2;  // streamed row box: 32 dims, 64 B rows
constexpr uint32_t kQBoxBytes = kTcQ * 32 * 2;       // streamed query box
constexpr int kMaxStages = 8;
constexpr uint32_t kTcSmem = 232448;  // 227 KB
constexpr float kNothing = -1e30f;    // a reference below every logit
constexpr float kEmpty = -2e30f;      // the logit of an empty slot: exp2 gives 0 against any

// Softmax sums of one (span, column half, query), in base 2 and relative to ref: over all
// scores but those of chunk `best`, whose own sums are b0, b1.
struct __align__(16) TcPart {
    float ref, e0, e1, b0, b1;
    int best;
    int pad[2];
};

struct TcDev {
    int n_rt;      // row tiles of this launch
    int n_kc;      // 32-dim chunks
    int n_qb;
    int n_q_pad;
    int n_stages;
    int chunk0;    // first chunk of this launch's rows
    const float* tab;  // [n_rt][256 factors | 256 offsets]
    float* mx;     // [chunk / kGroup][n_q_pad][kGroup] best logit of a chunk
    float* gx;     // [n_q_pad][g_pitch] best logit of a group
    int g_pitch;
    TcPart* part;  // [2 spans of a query block][128 n_qb] of this launch
    float* out;    // scores: of query 0 and this launch's row 0
    long long ldo;
    int n_q, n_rows;
    int vec;       // 1: out and ldo allow 32-byte stores
    int* err;
};

// The launch's tiles in the order (query block, row tile) are dealt out evenly: block c of G
// takes those from c T / G on, in spans of one query block each.
__host__ __device__ inline long long first_tile(long long tiles, int blocks, int c) {
    return c * tiles / blocks;
}
// The block that takes tile x.
__host__ __device__ inline int block_of(long long tiles, int blocks, long long x) {
    return (int)(((x + 1) * blocks - 1) / tiles);
}
// Spans of query block qb.
__host__ __device__ inline int spans_of(long long tiles, int blocks, int n_rt, int qb) {
    return block_of(tiles, blocks, (long long)qb * n_rt + n_rt - 1) -
           block_of(tiles, blocks, (long long)qb * n_rt) + 1;
}

struct Span {
    long long pos, end;  // what is left of the block's tiles
    int qb, t0, t1;

    __device__ __forceinline__ Span(const TcDev& p) {
        const long long tiles = (long long)p.n_qb * p.n_rt;
        pos = first_tile(tiles, gridDim.x, blockIdx.x);
        end = first_tile(tiles, gridDim.x, blockIdx.x + 1);
    }
    __device__ __forceinline__ bool next(const TcDev& p) {
        if (pos >= end) return false;
        qb = (int)(pos / p.n_rt);
        t0 = (int)(pos - (long long)qb * p.n_rt);
        t1 = (int)min((long long)p.n_rt, t0 + (end - pos));
        pos += t1 - t0;
        return true;
    }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
        : "memory");
}

// One whole 32-byte sector.
__device__ __forceinline__ void store8(float* p, const float (&a)[4], const float (&b)[4]) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(a[0]),
                 "f"(a[1]), "f"(a[2]), "f"(a[3]), "f"(b[0]), "f"(b[1]), "f"(b[2]), "f"(b[3])
                 : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// ---------------------------------------------------------------------------
// 1: operands
// ---------------------------------------------------------------------------
struct PrepareArgs {
    const void* q;
    int q_type;
    long long ldq;
    int n_q, n_q_pad;  // queries; rows of `parts` (0: the queries are there already)
    __half* parts;     // [n_q_pad][hi dim_pad | lo dim_pad]
    RegDev r;
    int row0, n_rows, n_pad;  // registry rows to expand, and the rows of `rows`
    float factor;             // what a row's scale is multiplied with
    __half* rows;             // [n_pad][dim_pad]
    float* tab;
    int* err;
};

constexpr int kExpandRows = 4;

// The first n_q_pad / 8 blocks take a query a warp; in the others a thread takes 8 dimensions
// of kExpandRows rows, rows past n_rows being zero and empty. L2 / HBM bound: bits / 8 bytes in
// and 2 bytes out a dimension of a row; 8192 queries and 100,000 8-bit rows of 256 dimensions
// take 14 us.
template <int BITS>
__global__ void __launch_bounds__(256)
registry_prepare_kernel(const __grid_constant__ PrepareArgs p) {
    const int n_split = p.n_q_pad / 8, dim_pad = p.r.dim_pad;
    if ((int)blockIdx.x < n_split) {
        const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
        if (blockIdx.x == 0 && threadIdx.x == 0) *p.err = 0;
        __half* hi = p.parts + (long long)row * 2 * dim_pad;
        split_query(p.q, p.q_type, (long long)row * p.ldq, p.r.dim, dim_pad, row < p.n_q,
                    StoreParts{hi, hi + dim_pad});
        return;
    }
    const int per = dim_pad / 8, in_block = 256 / per;  // threads a row, rows a block
    const int ty = threadIdx.x / per, d0 = (threadIdx.x - ty * per) * 8;
    const int first = (blockIdx.x - n_split) * (in_block * kExpandRows) + ty;
    if (ty >= in_block) return;
    // all loads first
    uint2 c[kExpandRows];
    uint32_t s16[kExpandRows];
    float scale[kExpandRows];
#pragma unroll
    for (int i = 0; i < kExpandRows; ++i) {
        const int row = first + i * in_block;
        c[i] = make_uint2(0x80808080u, 0x80808080u);
        s16[i] = 0u;
        scale[i] = __int_as_float(0x7FC00000);
        if (row >= p.n_rows) continue;
        const long long slot = (long long)p.row0 + row;
        const uint8_t* codes = p.r.codes + slot * p.r.row_bytes;
        if constexpr (BITS == 8) {
            c[i] = *reinterpret_cast<const uint2*>(codes + d0);
        } else {
            c[i].x = *reinterpret_cast<const uint32_t*>(codes + d0 / 2);
            s16[i] = p.r.group[slot * p.r.gpitch + d0 / 32];
        }
        if (d0 == 0) scale[i] = p.r.scale[slot];
    }
#pragma unroll
    for (int i = 0; i < kExpandRows; ++i) {
        const int row = first + i * in_block;
        if (row >= p.n_pad) break;
        uint32_t h[4];
        if constexpr (BITS == 8) {
            widen8(c[i].x, h[0], h[1]);
            widen8(c[i].y, h[2], h[3]);
        } else {
            const uint32_t s = h2_sub(s16[i] * 0x00010001u | 0x64006400u, 0x64006400u);
            widen4(c[i].x, s, h2_fma(s, 0xD480D480u, 0u), h);
        }
        *reinterpret_cast<uint4*>(p.rows + (long long)row * dim_pad + d0) =
            make_uint4(h[0], h[1], h[2], h[3]);
        if (d0 == 0) {
            const bool live = scale[i] == scale[i];
            float* t = p.tab + (long long)(row / kTcRows) * (2 * kTcRows) + row % kTcRows;
            t[0] = live ? scale[i] * p.factor : 0.0f;
            t[kTcRows] = live ? 0.0f : kEmpty;
        }
    }
}

// ---------------------------------------------------------------------------
// 2: scores, or chunk maxima and softmax sums
// ---------------------------------------------------------------------------
struct TcSums {
    float ref, e0, e1, bm, b0, b1;
    int best;
    __device__ __forceinline__ void reset() {
        ref = bm = kNothing;
        e0 = e1 = b0 = b1 = 0.0f;
        best = -1;
    }
};

// Four chunks of 8 logits of one query; their best logits. Packed f32 pairs halve the
// multiply-adds; a score costs 4 instructions and one exp2 (16 a cycle an SM: the epilogue's
// bound, half of the products' time at 256 dimensions).
__device__ __forceinline__ void add_chunks(const uint32_t (&v)[32], const float* tab, int chunk,
                                           TcSums& s, float (&top)[4]) {
    f2 y[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(tab + 4 * i);
        const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(tab + kTcRows + 4 * i);
        y[2 * i] = fma2(pack2(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1])), f.x, o.x);
        y[2 * i + 1] =
            fma2(pack2(__uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3])), f.y, o.y);
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        top[h] = kEmpty;
#pragma unroll
        for (int i = 4 * h; i < 4 * h + 4; ++i) {
            float a, b;
            unpack2(y[i], a, b);
            top[h] = fmaxf(fmaxf(top[h], a), b);
        }
    }
    const float all = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    if (all > s.ref + 60.0f) {
        // keep every exp2 below 2^60: rarely after a thread's first chunk
        const float d = s.ref - all, f = ex2(d);
        s.e1 = f * (s.e1 + s.e0 * d);
        s.e0 *= f;
        s.b1 = f * (s.b1 + s.b0 * d);
        s.b0 *= f;
        s.ref = all;
    }
    const f2 minus = pack2(-s.ref, -s.ref);
    f2 sum0[4], sum1[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        sum0[h] = sum1[h] = 0ull;
#pragma unroll
        for (int i = 4 * h; i < 4 * h + 4; ++i) {
            const f2 t = add2(y[i], minus);
            float a, b;
            unpack2(t, a, b);
            const f2 e = pack2(ex2(a), ex2(b));
            sum0[h] = add2(sum0[h], e);
            sum1[h] = fma2(e, t, sum1[h]);
        }
    }
    if (all <= s.bm) {
        // no chunk of these is the best so far
        float a, b, c, d;
        unpack2(add2(add2(sum0[0], sum0[1]), add2(sum0[2], sum0[3])), a, b);
        unpack2(add2(add2(sum1[0], sum1[1]), add2(sum1[2], sum1[3])), c, d);
        s.e0 += a + b;
        s.e1 += c + d;
        return;
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        float a, b, c, d;
        unpack2(sum0[h], a, b);
        unpack2(sum1[h], c, d);
        const float n0 = a + b, n1 = c + d;
        const bool first = top[h] > s.bm;  // the earlier chunk stays on equal scores
        s.e0 += first ? s.b0 : n0;
        s.e1 += first ? s.b1 : n1;
        s.b0 = first ? n0 : s.b0;
        s.b1 = first ? n1 : s.b1;
        s.bm = first ? top[h] : s.bm;
        s.best = first ? chunk + h : s.best;
    }
}

// 32 scores of one query to its row of the output; `left` of them inside the registry.
__device__ __forceinline__ void put_scores(const uint32_t (&v)[32], const float* tab, float* out,
                                           int left, bool vec) {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            o[j] = tab[kTcRows + i + j] < 0.0f ? -INFINITY
                                               : __uint_as_float(v[i + j]) * tab[i + j];
        if (vec && i + 8 <= left) {
            const float a[4] = {o[0], o[1], o[2], o[3]}, b[4] = {o[4], o[5], o[6], o[7]};
            store8(out + i, a, b);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < left) out[i + j] = o[j];
        }
    }
}

// RES: query parts resident in shared memory for a whole span (2: both, 1: the high part, 0:
// none); the others are streamed beside the rows, 32 dimensions a stage. Bound by the tensor
// pipe and the power it draws: 8192 queries x 100,000 rows x 256 dimensions, both parts (848
// GFLOP), take 579 us, 1.46 PFLOP/s; 4096 x 50,001 x 512 (RES 1) 315 us, 1.33 PFLOP/s.
template <int RES, bool STORE>
__global__ void __launch_bounds__(kTcThreads, 1)
registry_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmS,
                   const __grid_constant__ CUtensorMap tmR, const __grid_constant__ TcDev p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_u32 = smem_u32(smem_raw);
    const uint32_t base = (raw_u32 + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw_u32);
    constexpr uint32_t stage_bytes = kRowBoxBytes + (2 - RES) * kQBoxBytes;
    const int n_c64 = p.n_kc / 2;
    const uint32_t q_bytes = (uint32_t)RES * n_c64 * kResBytes;
    const uint32_t stage0 = q_bytes;
    const uint32_t tab0 = stage0 + p.n_stages * stage_bytes;
    const uint32_t bar0 = tab0 + kTabs * kTabBytes;
    const uint32_t bar_full = base + bar0;
    const uint32_t bar_empty = bar_full + 8 * kMaxStages;
    const uint32_t bar_tfull = bar_empty + 8 * kMaxStages;
    const uint32_t bar_tempty = bar_tfull + 16;
    const uint32_t bar_qfull = bar_tempty + 16;
    const uint32_t bar_qempty = bar_qfull + 8;
    const uint32_t bar_tabfull = bar_qempty + 8;
    const uint32_t bar_tabempty = bar_tabfull + 8 * kTabs;
    uint32_t* tmem_slot =
        reinterpret_cast<uint32_t*>(smem + bar0 + 8 * (2 * kMaxStages + 6 + 2 * kTabs));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.n_stages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_tfull + 8 * a, 1);
            mbar_init(bar_tempty + 8 * a, 8);
        }
        for (int a = 0; a < kTabs; ++a) {
            mbar_init(bar_tabfull + 8 * a, 1);
            mbar_init(bar_tabempty + 8 * a, 8);
        }
        mbar_init(bar_qfull, 1);
        mbar_init(bar_qempty, 1);
        *abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async_smem();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmR);
        if (RES > 0) tma_prefetch_desc(&tmQ);
        if (RES < 2) tma_prefetch_desc(&tmS);
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer ----------------
            pdl_wait();  // for the operands; every other role's first read follows its loads
            uint32_t stage = 0, phase = 0, qphase = 0, tab = 0, tab_phase = 0;
            bool ok = true;
            Span span(p);
            while (ok && span.next(p)) {
                const int qb = span.qb;
                if constexpr (RES > 0) {
                    // the previous span's MMAs are done with the resident parts
                    if (!mbar_wait(bar_qempty, qphase ^ 1, p.err, VDB_ERR_TIMEOUT_EMPTY,
                                   abort_flag)) {
                        ok = false;
                        break;
                    }
                    qphase ^= 1;
                    mbar_arrive_expect_tx(bar_qfull, q_bytes);
                    // the parts are neighbours along the rows of [hi | lo]
                    for (int c = 0; c < RES * n_c64; ++c)
                        tma_load_2d(base + (uint32_t)c * kResBytes, &tmQ, bar_qfull, c * 64,
                                    qb * kTcQ);
                }
                for (int t = span.t0; t < span.t1 && ok; ++t) {
                    if (!mbar_wait(bar_tabempty + 8 * tab, tab_phase ^ 1, p.err,
                                   VDB_ERR_TIMEOUT_EMPTY, abort_flag)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(bar_tabfull + 8 * tab, kTabBytes);
                    bulk_load(base + tab0 + tab * kTabBytes, p.tab + (long long)t * (2 * kTcRows),
                              kTabBytes, bar_tabfull + 8 * tab);
                    if (++tab == kTabs) {
                        tab = 0;
                        tab_phase ^= 1;
                    }
                    for (int c = 0; c < p.n_kc; ++c) {
                        if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1, p.err,
                                       VDB_ERR_TIMEOUT_EMPTY, abort_flag)) {
                            ok = false;
                            break;
                        }
                        const uint32_t dst = base + stage0 + stage * stage_bytes;
                        mbar_arrive_expect_tx(bar_full + 8 * stage, stage_bytes);
                        tma_load_2d(dst, &tmR, bar_full + 8 * stage, c * 32, t * kTcRows);
                        if constexpr (RES == 0)
                            tma_load_2d(dst + kRowBoxBytes, &tmS, bar_full + 8 * stage, c * 32,
                                        qb * kTcQ);
                        if constexpr (RES < 2)
                            tma_load_2d(dst + kRowBoxBytes + (1 - RES) * kQBoxBytes, &tmS,
                                        bar_full + 8 * stage, (p.n_kc + c) * 32, qb * kTcQ);
                        if (++stage == (uint32_t)p.n_stages) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                }
            }
            if (!ok) {
                // copies still in flight land before the block gives its memory back
                for (int i = 0; i < p.n_stages; ++i)
                    mbar_wait_drain(bar_full + 8 * i, phase, 20000000ull);
                for (int i = 0; i < kTabs; ++i)
                    mbar_wait_drain(bar_tabfull + 8 * i, tab_phase, 20000000ull);
                mbar_wait_drain(bar_qfull, qphase ^ 1, 20000000ull);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // ---------------- MMA issuer ----------------
            const uint32_t idesc = umma_idesc_f16(kTcQ, kTcRows);
            uint32_t stage = 0, phase = 0, qphase = 0, acc = 0, acc_phase = 0;
            bool ok = true, issued = false;
            const uint64_t q_desc = umma_sdesc(base, 128);
            const uint64_t s_desc = umma_sdesc(base + stage0, 64);
            Span span(p);
            while (ok && span.next(p)) {
                if constexpr (RES > 0) {
                    if (!mbar_wait(bar_qfull, qphase, p.err, VDB_ERR_TIMEOUT_FULL, abort_flag)) {
                        ok = false;
                        break;
                    }
                    qphase ^= 1;
                    tc_fence_after();
                }
                for (int t = span.t0; t < span.t1 && ok; ++t) {
                    if (!mbar_wait(bar_tempty + 8 * acc, acc_phase ^ 1, p.err,
                                   VDB_ERR_TIMEOUT_TEMPTY, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem_base + acc * kTcRows;
                    for (int c = 0; c < p.n_kc; ++c) {
                        if (!mbar_wait(bar_full + 8 * stage, phase, p.err, VDB_ERR_TIMEOUT_FULL,
                                       abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint64_t b = s_desc + (uint64_t)(stage * (stage_bytes >> 4));
                        const uint64_t qs = b + (kRowBoxBytes >> 4);
                        const uint64_t qr = q_desc + (uint64_t)((c >> 1) * (kResBytes >> 4)) +
                                            (uint64_t)((c & 1) * 4);
                        const uint64_t hi = RES > 0 ? qr : qs;
                        const uint64_t lo = RES == 2 ? qr + (uint64_t)(n_c64 * (kResBytes >> 4))
                                                     : qs + (1 - RES) * (kQBoxBytes >> 4);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            umma_f16(d, hi + 2 * k, b + 2 * k, idesc, (c | k) ? 1u : 0u);
                            umma_f16(d, lo + 2 * k, b + 2 * k, idesc, 1u);
                        }
                        umma_commit(bar_empty + 8 * stage);
                        issued = true;
                        if (++stage == (uint32_t)p.n_stages) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                    if (!ok) break;
                    umma_commit(bar_tfull + 8 * acc);
                    if (++acc == 2) {
                        acc = 0;
                        acc_phase ^= 1;
                    }
                }
                if (!ok) break;
                if constexpr (RES > 0) umma_commit(bar_qempty);
            }
            if (!ok && issued) {
                const uint32_t last = (stage + p.n_stages - 1) % p.n_stages;
                mbar_wait_drain(bar_empty + 8 * last, phase ^ (stage == 0 ? 1u : 0u), 20000000ull);
            }
        }
    } else if (warp >= 4) {
        // ---------------- epilogue: thread = query (TMEM lane), half of the columns -----
        const int quad = warp & 3, half = (warp - 4) >> 2;
        uint32_t acc = 0, acc_phase = 0, tab = 0, tab_phase = 0;
        bool ok = true;
        Span span(p);
        while ((ok || STORE) && span.next(p)) {
            const int q = span.qb * kTcQ + quad * 32 + lane;
            TcSums s;
            s.reset();
            for (int t = span.t0; t < span.t1; ++t) {
                if (ok && (!mbar_wait(bar_tabfull + 8 * tab, tab_phase, p.err,
                                      VDB_ERR_TIMEOUT_TFULL, abort_flag) ||
                           !mbar_wait(bar_tfull + 8 * acc, acc_phase, p.err,
                                      VDB_ERR_TIMEOUT_TFULL, abort_flag)))
                    ok = false;
                if (!ok) {
                    // a wait ran out: no scores are better than what the memory held (a
                    // posterior's last kernel sees the error word)
                    if constexpr (!STORE) break;
                    const int col = t * kTcRows + half * (kTcRows / 2);
                    for (int i = 0; q < p.n_q && i < kTcRows / 2 && col + i < p.n_rows; ++i)
                        p.out[(long long)q * p.ldo + col + i] = __int_as_float(0x7FC00000);
                    continue;
                }
                tc_fence_after();
                const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + acc * kTcRows +
                                       (uint32_t)(half * (kTcRows / 2));
                const float* tb = reinterpret_cast<const float*>(smem + tab0 + tab * kTabBytes) +
                                  half * (kTcRows / 2);
                const int group = p.chunk0 / kGroup + 2 * t + half, chunk = group * kGroup;
                const long long at = (long long)group * p.n_q_pad + q;
                float best = kEmpty;
#pragma unroll 1
                for (int c = 0; c < 4; c += 2) {
                    uint32_t v[2][32];
                    __syncwarp();  // tcgen05.ld is warp-collective: reconverge first
                    tmem_ld_32x32b_x32_nowait(taddr + (uint32_t)(c * 32), v[0]);
                    tmem_ld_32x32b_x32_nowait(taddr + (uint32_t)(c * 32 + 32), v[1]);
                    tmem_wait_ld();
                    tmem_regs_ready(v[0]);
                    tmem_regs_ready(v[1]);
                    if (c == 2) {
                        // the accumulator is free before its last 64 columns are summed
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar_tempty + 8 * acc);
                    }
                    if constexpr (STORE) {
                        if (q < p.n_q) {
                            const int col = t * kTcRows + half * (kTcRows / 2) + c * 32;
                            float* out = p.out + (long long)q * p.ldo + col;
                            put_scores(v[0], tb + c * 32, out, p.n_rows - col, p.vec);
                            put_scores(v[1], tb + c * 32 + 32, out + 32, p.n_rows - col - 32, p.vec);
                        }
                        continue;
                    }
                    float ta[4], tb_[4];
                    add_chunks(v[0], tb + c * 32, chunk + 4 * c, s, ta);
                    add_chunks(v[1], tb + c * 32 + 32, chunk + 4 * c + 4, s, tb_);
                    store8(p.mx + at * kGroup + 4 * c, ta, tb_);
#pragma unroll
                    for (int h = 0; h < 4; ++h) best = fmaxf(best, fmaxf(ta[h], tb_[h]));
                }
                if constexpr (!STORE) p.gx[(long long)q * p.g_pitch + group] = best;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_tabempty + 8 * tab);
                if (++tab == kTabs) {
                    tab = 0;
                    tab_phase ^= 1;
                }
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
            if constexpr (STORE) continue;
            if (!ok) break;
            TcPart o;
            o.ref = s.ref, o.e0 = s.e0, o.e1 = s.e1, o.b0 = s.b0, o.b1 = s.b1, o.best = s.best;
            o.pad[0] = o.pad[1] = 0;
            const int nth = blockIdx.x - block_of((long long)p.n_qb * p.n_rt, gridDim.x,
                                                  (long long)span.qb * p.n_rt);
            p.part[(long long)(2 * nth + half) * (p.n_qb * kTcQ) + q] = o;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ---------------------------------------------------------------------------
// 3: the answer
// ---------------------------------------------------------------------------
constexpr int kHotCand = 128;  // groups, and chunks, that may reach the bound (L <= 68)

__device__ __forceinline__ bool is_live(float v) { return v > kNothing; }

// The best L chunks of one query by (best logit, lower chunk), by one warp (L rounded up to
// even: two make a product's 16 rows), in any order; returns their number. gx: the query's group
// maxima; mx: its chunk maxima of group g at mx + g * m_pitch; span: more than two logits
// differ. The L-th largest of 128 (for L <= 12: 32) maxima of disjoint sets of groups bounds the
// L-th best chunk's from below, and the few groups and chunks that reach it are collected.
__device__ __forceinline__ int hot_chunks(const float* __restrict__ gx,
                                          const float* __restrict__ mx, long long m_pitch,
                                          int n_groups, int L, float span, int* chunks, float* cs,
                                          int* ci, int* hg, int* count) {
    const int lane = threadIdx.x & 31;
    constexpr unsigned full = 0xffffffffu;
    if (lane < 2) count[lane] = 0;
    // groups i .. i + 3; the row's pitch is a multiple of 4, n_groups of 2
    const auto four = [&](int i) {
        float4 v = *reinterpret_cast<const float4*>(gx + i);
        if (i + 2 >= n_groups) v.z = v.w = kEmpty;
        return v;
    };
    float4 m = make_float4(kEmpty, kEmpty, kEmpty, kEmpty);
#pragma unroll 4
    for (int i = lane * 4; i < n_groups; i += 128) {
        const float4 v = four(i);
        m = make_float4(fmaxf(m.x, v.x), fmaxf(m.y, v.y), fmaxf(m.z, v.z), fmaxf(m.w, v.w));
    }
    const auto key = [](float v) { return is_live(v) ? key_of(v) : 0u; };
    uint32_t low;
    if (L <= 12) {
        low = lth_lane_key(key(fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w))), L);
    } else {
        const uint32_t all[4] = {key(m.x), key(m.y), key(m.z), key(m.w)};
        low = lth_key<4>(all, L);
    }
    // fewer than L sets hold anything: everything alive
    const float bound = low == 0 ? nextafterf(kNothing, 0.0f) : from_key(low);
    __syncwarp();
#pragma unroll 2
    for (int i = lane * 4; i < n_groups; i += 128) {
        const float4 v = four(i);
        if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= bound)) continue;
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (e[j] >= bound) {
                const int pos = atomicAdd(count, 1);
                if (pos < kHotCand) hg[pos] = i + j;
            }
    }
    __syncwarp();
    // the chunks of the groups found, four at a time; of all groups when they are too many
    constexpr int kQuads = kGroup / 4;
    const int ng = count[0];
    const bool some = ng <= kHotCand;
    const int n_quad = (some ? ng : n_groups) * kQuads;
    const auto quad_at = [&](int g, int e) {
        return __ldg(reinterpret_cast<const float4*>(mx + g * m_pitch + e % kQuads * 4));
    };
    const auto group_of = [&](int e) { return some ? hg[e / kQuads] : e / kQuads; };
    const auto reach = [&](float least) {
        int c = 0;
        for (int e = lane; e < n_quad; e += 32) {
            const float4 v = quad_at(group_of(e), e);
            c += (v.x >= least) + (v.y >= least) + (v.z >= least) + (v.w >= least);
        }
        return (int)__reduce_add_sync(full, c);
    };
    const auto collect = [&](float least) {
        if (lane == 0) count[1] = 0;
        __syncwarp();
        for (int e = lane; e < n_quad; e += 32) {
            const int g = group_of(e);
            const float4 v = quad_at(g, e);
            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (x[j] >= least) {
                    const int pos = atomicAdd(count + 1, 1);
                    if (pos < kHotCand) cs[pos] = x[j], ci[pos] = g * kGroup + e % kQuads * 4 + j;
                }
        }
        __syncwarp();
        return count[1];
    };
    L += L & 1;
    int cnt = some ? collect(bound) : kHotCand + 1;
    float tie = 0.0f;  // where no bound separates L to kHotCand chunks: the L-th best logit
    if (cnt > kHotCand) {
        // bisection in the logits for a bound that L to kHotCand chunks reach
        float lo = bound, hi = fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w));
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) hi = fmaxf(hi, __shfl_xor_sync(full, hi, o));
        lo = fmaxf(lo, -fabsf(hi) - span);  // below every logit
        while (true) {
            const float mid = 0.5f * lo + 0.5f * hi;
            const bool last = !(mid > lo && mid < hi);
            const int c = reach(last ? hi : mid);
            if (c >= L && c <= kHotCand) {
                cnt = collect(last ? hi : mid);
                break;
            }
            if (last) {
                tie = c >= L ? hi : lo;
                break;
            }
            if (c >= L)
                lo = mid;
            else
                hi = mid;
        }
    }
    if (cnt <= L) {
        for (int e = lane; e < cnt; e += 32) chunks[e] = ci[e];
    } else if (cnt <= kHotCand) {
        for (int e = lane; e < cnt; e += 32) {
            const float s = cs[e];
            const int c = ci[e];
            int rank = 0;
            for (int i = 0; i < cnt; ++i) rank += ahead(cs[i], ci[i], s, c) ? 1 : 0;
            if (rank < L) chunks[rank] = c;
        }
        cnt = L;
    } else {
        // many chunks tie: those above, and the first of the equal ones in chunk order
        const int above = reach(nextafterf(tie, INFINITY));
        int n_above = 0, n_equal = 0;
        for (int e0 = 0; e0 < n_groups * kQuads && n_above + n_equal < L; e0 += 32) {
            const int e = e0 + lane, g = e / kQuads;
            float4 v = make_float4(kEmpty, kEmpty, kEmpty, kEmpty);
            if (e < n_groups * kQuads) v = quad_at(g, e);
            const float x[4] = {v.x, v.y, v.z, v.w};
            // this lane's (above, equal) counts, packed, and those of the lanes before it
            int own = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) own += x[j] > tie ? 1 << 16 : x[j] == tie ? 1 : 0;
            int sum = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(full, sum, o);
                sum += lane >= o ? y : 0;
            }
            int pa = n_above + ((sum - own) >> 16), pe = n_equal + ((sum - own) & 0xFFFF);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = g * kGroup + e % kQuads * 4 + j;
                if (x[j] > tie) {
                    if (pa < L) chunks[pa] = c;
                    ++pa;
                } else if (x[j] == tie) {
                    if (pe < L - above) chunks[above + pe] = c;
                    ++pe;
                }
            }
            sum = __shfl_sync(full, sum, 31);
            n_above += sum >> 16;
            n_equal = min(n_equal + (sum & 0xFFFF), L - above);
        }
        cnt = min(L, n_above + n_equal);
    }
    __syncwarp();
    return cnt;
}

// Candidates rescored at most: L, up to a whole number of fours with the label's.
__host__ __device__ constexpr int answer_size(int L) { return L / 4 * 4 + 3; }

struct AnswerArgs {
    MergeArgs m;
    int q0, n_q;  // queries of this launch
    const __half* qs;
    const float *mx, *gx;
    int n_groups, g_pitch;
    const TcPart* part;  // [segment][2 n_span][128 n_qb]
    int n_seg, n_span, n_q_pad, L;
    int n_qb, sms, seg_rt, last_rt;  // tiles of a segment, of the last one
    float s2;
    const int* err;
};

// One block of 1 to 8 warps per query. With many queries one warp each: the steps are short
// and depend on one another, so warps of other queries are what hides their latencies; a few
// hundred queries are spread over more warps. Shared memory: the query, the scores and slots
// of the chunks, the selection's lists. 98 us for 8192 queries, 100,000 8-bit rows of 256
// dimensions and k = 5; of a block's 50 us 20 are the chunks' rows (gathers of 256 bytes from L2,
// 4.4 TB/s in all), 12 the maxima, 7 the f64 products.
template <int BITS>
__global__ void __launch_bounds__(256, 4)
registry_answer_kernel(const __grid_constant__ AnswerArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ double ex[answer_size(kRegMaxK + kRegExtra) + 1];
    __shared__ double s_qq;
    __shared__ float bs[answer_size(kRegMaxK + kRegExtra)];
    __shared__ int bi[answer_size(kRegMaxK + kRegExtra)], rank[answer_size(kRegMaxK + kRegExtra)];
    __shared__ int hot[kRegMaxK + kRegExtra];
    __shared__ float hot_s[kHotCand];
    __shared__ int hot_i[kHotCand], hot_g[kHotCand], hot_n[2], s_hot;
    const MergeArgs& p = a.m;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n_warps = blockDim.x / 32;
    const int row = blockIdx.x;  // of this launch
    const int qi = a.q0 + row;   // of the call
    const int L = a.L, most = (L + 1) / 2 * 2 * kChunk;
    double* qv = reinterpret_cast<double*>(smem);
    float* sc = reinterpret_cast<float*>(qv + p.r.dim_pad);
    int* slot = reinterpret_cast<int*>(sc + most);
    float* list_s = reinterpret_cast<float*>(slot + most);
    const int cap = answer_size(L);
    int* list_i = reinterpret_cast<int*>(list_s + 2 * cap);
    if (warp == n_warps - 1) {
        const double s = stage_query(p, qi, qv);
        if (lane == 0) s_qq = s;
    }
    const int label = label_of(p, qi);
    pdl_wait();
    if (warp == 0) {
        const int n = hot_chunks(a.gx + (long long)row * a.g_pitch, a.mx + (long long)row * kGroup,
                                 (long long)a.n_q_pad * kGroup, a.n_groups, L, 2.1f * a.s2, hot, hot_s,
                                 hot_i, hot_g, hot_n);
        if (lane == 0) s_hot = n;
    }
    __syncthreads();
    const int n_hot = s_hot, n_ent = n_hot * kChunk;
    const int n_c = p.r.dim_pad / 64;
    const uint64_t policy = code_policy(0);
    const __half* part_of = a.qs + ((long long)row * 2 + (g & 1)) * p.r.dim_pad + 16 * t;
    // 16 rows a product: two chunks
    for (int tile = warp; 2 * tile < n_hot; tile += n_warps) {
        const bool two = 2 * tile + 1 < n_hot;
        const int ra = hot[2 * tile] * kChunk + g, rb = two ? hot[2 * tile + 1] * kChunk + g : ra;
        const bool ina = ra < p.n_rows, inb = two && rb < p.n_rows;
        const long long la = min(ra, p.n_rows - 1), lb = min(rb, p.n_rows - 1);
        const float sa = p.r.scale[la], sb = p.r.scale[lb];
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c0 = 0; c0 < n_c; c0 += 4) {
            RowFrag<BITS> f;
            f.load(p.r, la, lb, c0, n_c, t, policy);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (c0 + u >= n_c) break;
                uint32_t fa[8], fb[8];
                f.widen(u, t, fa, fb);
                uint4 b0 = make_uint4(0u, 0u, 0u, 0u), b1 = b0;
                if (g < 2) {  // column 0: the high part, 1: the low part
                    const uint4* qb = reinterpret_cast<const uint4*>(part_of + (c0 + u) * 64);
                    b0 = __ldg(qb);
                    b1 = __ldg(qb + 1);
                }
                mma_16816(acc, fa[0], fb[0], fa[1], fb[1], b0.x, b0.y);
                mma_16816(acc, fa[2], fb[2], fa[3], fb[3], b0.z, b0.w);
                mma_16816(acc, fa[4], fb[4], fa[5], fb[5], b1.x, b1.y);
                mma_16816(acc, fa[6], fb[6], fa[7], fb[7], b1.z, b1.w);
            }
        }
        if (t == 0) {
            const int at = tile * 2 * kChunk + g;
            sc[at] = ina && sa == sa ? (acc[0] + acc[1]) * (sa * (1.0f / kQScale)) : -INFINITY;
            slot[at] = ra;
            if (two) {
                sc[at + kChunk] =
                    inb && sb == sb ? (acc[2] + acc[3]) * (sb * (1.0f / kQScale)) : -INFINITY;
                slot[at + kChunk] = rb;
            }
        }
    }
    __syncthreads();
    // n_ent <= 544: mostly one warp's selection of at most 256
    if (n_ent <= 256) {
        if (warp == 0)
            warp_select<8>(sc, slot, 0, n_ent, L, cap, a.s2, bs, bi);
    } else {
        for (int part = warp; part < 2; part += n_warps)
            warp_select<16>(sc + part * kPart, slot + part * kPart, 0,
                            max(0, min(kPart, n_ent - part * kPart)), L, cap, a.s2,
                            list_s + part * cap, list_i + part * cap);
        __syncthreads();
        if (warp == 0)
            warp_select<8>(list_s, list_i, 0, 2 * cap, L, cap, a.s2, bs, bi);
    }
    __syncthreads();
    int nb = 0;
    for (int i = lane; i < cap; i += 32) nb += bi[i] >= 0 ? 1 : 0;
    nb = __reduce_add_sync(0xffffffffu, nb);
    const double qq = s_qq;
    rescore(p, qv, qq, bi, nb, label, ex);
    __syncthreads();
    rank_candidates(ex, bi, nb, rank);
    __syncthreads();
    if (warp != 0) return;
    // a wait that ran out upstream leaves no numbers to trust
    const bool bad = !finite(qq) || *a.err != 0;
    const int top = first_candidate(rank, nb);
    double M = 0.0;
    float E = 0.0f, S = 0.0f;
    if (nb > 0 && !bad) {
        M = ex[top];
        const double T = (double)p.temperature, M2 = M * (double)a.s2;
        const int ct = bi[top] / kChunk;
        bool hit = false;  // the top score's chunk was kept apart from the sums
        for (int i = lane; i < a.n_seg * 2 * a.n_span; i += 32) {
            const int sg = i / (2 * a.n_span), nth = (i - sg * 2 * a.n_span) / 2;
            const int n_rt = sg == a.n_seg - 1 ? a.last_rt : a.seg_rt;
            const long long tiles = (long long)a.n_qb * n_rt;
            if (nth >= spans_of(tiles, (int)min(tiles, (long long)a.sms), n_rt, row / kTcQ))
                continue;
            const TcPart o = a.part[(long long)i * (a.n_qb * kTcQ) + row];
            if (!is_live(o.ref)) continue;
            const float d = (float)((double)o.ref - M2), f = exp2f(d);
            const bool mine = o.best == ct;
            hit |= mine;
            const float e0 = o.e0 + (mine ? 0.0f : o.b0), e1 = o.e1 + (mine ? 0.0f : o.b1);
            E += f * e0;
            S += 0.69314718f * (f * (e1 + e0 * d));
        }
        if (__any_sync(0xffffffffu, hit)) {
            for (int i = lane; i < n_ent; i += 32) {
                if (hot[i / kChunk] != ct || slot[i] == bi[top] || !(sc[i] > -INFINITY)) continue;
                const float d = (float)(T * ((double)sc[i] - M)), e = expf(d);
                E += e;
                S += e * d;
            }
        } else if (lane == 0) {
            // another chunk's score rounded to the same or a higher f32: the top score is
            // inside the sums, which are at least about as large
            const float d = (float)(T * ((double)bs[top] - M)), e = expf(d);
            E -= e;
            S -= e * d;
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
            E += __shfl_xor_sync(0xffffffffu, E, o);
            S += __shfl_xor_sync(0xffffffffu, S, o);
        }
        E = fmaxf(E, 0.0f);
    }
    write_posterior(p, qi, bi, ex, nb, rank, bad, label, M, (double)E, (double)S);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr size_t answer_smem(int dim_pad, int L) {
    return (size_t)dim_pad * 8 + (size_t)((L + 1) / 2 * 2) * kChunk * 8 +
           (size_t)2 * answer_size(L) * 8;
}
// with the kernel's 3.3 KB of static shared memory below what needs an opt-in
static_assert(answer_smem(kRegMaxDim, kRegMaxK + kRegExtra) <= 40 * 1024, "");

struct TcPlan {
    int dim_pad, L;
    int res, n_stages;
    int qbatch;             // queries per pass over the registry (a multiple of 128)
    long long seg_rows;     // rows expanded at a time (a multiple of 256)
    int n_seg;              // segments
    long long n_chunks;
    int g_pitch;
    size_t q_b, row_b, tab_b, mx_b, gx_b, part_b, total;
};

// Spans that a query block of n_qb is dealt out to at most: it is T / n_qb tiles of which a
// block takes T / SMs. (n_qb times this is at most SMs + 2 n_qb.)
int most_spans(int n_qb, long long n_rt) {
    return (int)std::min<long long>((num_sms() + n_qb - 1) / n_qb + 1, n_rt);
}

// k < 0: scores, which need neither maxima nor partials
TcPlan tc_plan(int n_rows, int n_q, int dim, int k) {
    TcPlan t{};
    const bool post = k >= 0;
    t.dim_pad = reg_dim_pad(dim);
    t.L = k + kRegExtra;
    // resident query parts: as many as leave three stages
    const uint32_t fixed = 1024 + kTabs * kTabBytes + 512;
    for (t.res = 2; t.res >= 0; --t.res) {
        const uint32_t q = (uint32_t)t.res * (t.dim_pad / 64) * kResBytes;
        const uint32_t st = kRowBoxBytes + (2 - t.res) * kQBoxBytes;
        if (q + fixed + 3 * st > kTcSmem) continue;
        t.n_stages = (int)std::min<uint32_t>(kMaxStages, (kTcSmem - fixed - q) / st);
        break;
    }
    const long long n_pad = ((long long)n_rows + kTcRows - 1) / kTcRows * kTcRows;
    t.n_chunks = n_pad / kChunk;
    // at most 256 MB of expanded rows and, over one batch of queries, 1 GB of maxima
    const long long most = (256LL << 20) / (t.dim_pad * 2) / kTcRows * kTcRows;
    t.n_seg = (int)((n_pad + most - 1) / most);
    t.seg_rows = (n_pad / kTcRows + t.n_seg - 1) / t.n_seg * kTcRows;
    t.n_seg = (int)((n_pad + t.seg_rows - 1) / t.seg_rows);
    const long long q_pad = ((long long)n_q + kTcQ - 1) / kTcQ * kTcQ;
    const long long fit = std::max<long long>(kTcQ, (1LL << 28) / t.n_chunks / kTcQ * kTcQ);
    t.qbatch = (int)std::min(post ? std::min(q_pad, fit) : q_pad, 1LL << 16);
    t.q_b = reg_up((size_t)t.qbatch * 2 * t.dim_pad * 2);
    t.row_b = reg_up((size_t)t.seg_rows * t.dim_pad * 2);
    t.tab_b = reg_up((size_t)(t.seg_rows / kTcRows) * kTabBytes);
    t.mx_b = post ? reg_up((size_t)t.n_chunks * t.qbatch * 4) : 0;
    t.part_b = post ? reg_up((size_t)t.n_seg * 2 * (num_sms() * kTcQ + 2 * t.qbatch) * sizeof(TcPart)) : 0;
    t.g_pitch = (int)((t.n_chunks / kGroup + 3) / 4 * 4);
    t.gx_b = post ? reg_up((size_t)t.g_pitch * t.qbatch * 4) : 0;
    t.total = t.q_b + t.row_b + t.tab_b + t.mx_b + t.gx_b + t.part_b + 256;
    return t;
}

bool map_2d(CUtensorMap* m, const void* ptr, long long width, long long rows, int box_w, int box_h,
            CUtensorMapSwizzle sw) {
    cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)width * 2};
    cuuint32_t box[2] = {(cuuint32_t)box_w, (cuuint32_t)box_h};
    cuuint32_t estr[2] = {1, 1};
    return encode_tiled_fn()(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(ptr), dims,
                             strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int RES, bool STORE>
cudaError_t launch_tc(const CUtensorMap& q, const CUtensorMap& s, const CUtensorMap& r,
                      const TcDev& d, cudaStream_t st) {
    static SmemOptIn opt_in;
    auto kern = registry_tc_kernel<RES, STORE>;
    cudaError_t e = opt_in.allow(kern, kTcSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)std::min<long long>((long long)d.n_qb * d.n_rt, num_sms()));
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = kTcSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, q, s, r, d);
}

template <int BITS>
cudaError_t launch_answer(const AnswerArgs& a, cudaStream_t st) {
    // about 28 warps an SM
    int warps = 8;
    while (warps > 1 && (long long)a.n_q * warps > 28LL * num_sms()) warps /= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)a.n_q);
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = answer_smem(a.m.r.dim_pad, a.L);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, registry_answer_kernel<BITS>, a);
}

}  // namespace

size_t registry_tc_work(int n_rows, int n_q, int dim, int k) {
    return tc_plan(n_rows, n_q, dim, k).total;
}

// Scores (k < 0: out, ldo) or posterior of all of m's queries.
cudaError_t registry_tc_run(const MergeArgs& m, int k, float* out, long long ldo, void* work,
                            cudaStream_t st) {
    const TcPlan t = tc_plan(m.n_rows, m.n_q, m.r.dim, k);
    const bool post = k >= 0;
    uint8_t* w = static_cast<uint8_t*>(work);
    __half* qs = reinterpret_cast<__half*>(w);
    w += t.q_b;
    __half* rows = reinterpret_cast<__half*>(w);
    w += t.row_b;
    float* tab = reinterpret_cast<float*>(w);
    w += t.tab_b;
    float* mx = reinterpret_cast<float*>(w);
    w += t.mx_b;
    float* gx = reinterpret_cast<float*>(w);
    w += t.gx_b;
    TcPart* part = reinterpret_cast<TcPart*>(w);
    w += t.part_b;
    int* err = reinterpret_cast<int*>(w);

    // The logits also rank the chunks, so their scale must keep them (and a row's factor, down
    // to s2 / (256 * 28448)) in f32's normal range. Below a temperature of 2^-40 every softmax
    // weight is 1 to within 2^-38, so the sums may take 2^-40 for it.
    const float s2 = post ? std::max(m.temperature, 0x1p-40f) * 1.4426950408889634f : 1.0f;
    CUtensorMap tq, ts, tr;
    if (!map_2d(&tq, qs, 2 * t.dim_pad, t.qbatch, 64, kTcQ, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !map_2d(&ts, qs, 2 * t.dim_pad, t.qbatch, 32, kTcQ, CU_TENSOR_MAP_SWIZZLE_64B) ||
        !map_2d(&tr, rows, t.dim_pad, t.seg_rows, 32, kTcRows, CU_TENSOR_MAP_SWIZZLE_64B))
        return cudaErrorInvalidValue;
    cudaError_t e = cudaSuccess;
    Batches batches{m.n_q, t.qbatch};
    for (int q0, nq; e == cudaSuccess && batches.next(q0, nq);) {
        const int n_qb = (nq + kTcQ - 1) / kTcQ;
        const int n_span = most_spans(n_qb, t.seg_rows / kTcRows);
        PrepareArgs pa{};
        pa.q = static_cast<const uint8_t*>(m.q) + (size_t)q0 * m.ldq * (m.q_type == kF32 ? 4 : 2);
        pa.q_type = m.q_type;
        pa.ldq = m.ldq;
        pa.n_q = nq;
        pa.parts = qs;
        pa.r = m.r;
        pa.factor = s2 * (1.0f / kQScale);
        pa.rows = rows;
        pa.tab = tab;
        pa.err = err;
        for (int sg = 0; sg < t.n_seg && e == cudaSuccess; ++sg) {
            pa.n_q_pad = sg == 0 ? n_qb * kTcQ : 0;
            pa.row0 = (int)(sg * t.seg_rows);
            pa.n_rows = (int)std::min<long long>(t.seg_rows, (long long)m.n_rows - pa.row0);
            const int n_rt = (pa.n_rows + kTcRows - 1) / kTcRows;
            pa.n_pad = n_rt * kTcRows;
            const int in_block = 256 / (t.dim_pad / 8);
            const int rows_block = in_block * kExpandRows;
            const unsigned grid =
                (unsigned)(pa.n_q_pad / 8 + (pa.n_pad + rows_block - 1) / rows_block);
            if (m.r.bits == 8)
                registry_prepare_kernel<8><<<grid, 256, 0, st>>>(pa);
            else
                registry_prepare_kernel<4><<<grid, 256, 0, st>>>(pa);
            e = cudaGetLastError();
            if (e != cudaSuccess) break;
            TcDev d{};
            d.n_rt = n_rt;
            d.n_kc = t.dim_pad / 32;
            d.n_qb = n_qb;
            d.n_q_pad = t.qbatch;
            d.n_stages = t.n_stages;
            d.chunk0 = pa.row0 / kChunk;
            d.tab = tab;
            d.mx = mx;
            d.gx = gx;
            d.g_pitch = t.g_pitch;
            d.part = part + (size_t)sg * 2 * n_span * n_qb * kTcQ;
            d.err = err;
            if (post) {
                e = t.res == 2   ? launch_tc<2, false>(tq, ts, tr, d, st)
                    : t.res == 1 ? launch_tc<1, false>(tq, ts, tr, d, st)
                                 : launch_tc<0, false>(tq, ts, tr, d, st);
            } else {
                d.out = out + (long long)q0 * ldo + pa.row0;
                d.ldo = ldo;
                d.n_q = nq;
                d.n_rows = pa.n_rows;
                d.vec = reinterpret_cast<uintptr_t>(d.out) % 32 == 0 && ldo % 8 == 0;
                e = t.res == 2   ? launch_tc<2, true>(tq, ts, tr, d, st)
                    : t.res == 1 ? launch_tc<1, true>(tq, ts, tr, d, st)
                                 : launch_tc<0, true>(tq, ts, tr, d, st);
            }
        }
        if (e != cudaSuccess || !post) continue;
        AnswerArgs a{};
        a.m = m;
        a.q0 = q0;
        a.n_q = nq;
        a.qs = qs;
        a.mx = mx;
        a.gx = gx;
        a.n_groups = (int)(t.n_chunks / kGroup);
        a.g_pitch = t.g_pitch;
        a.part = part;
        a.n_seg = t.n_seg;
        a.n_span = n_span;
        a.n_qb = n_qb;
        a.sms = num_sms();
        a.seg_rt = (int)(t.seg_rows / kTcRows);
        a.last_rt = (int)(((long long)m.n_rows - (t.n_seg - 1) * t.seg_rows + kTcRows - 1) / kTcRows);
        a.n_q_pad = t.qbatch;
        a.L = t.L;
        a.s2 = s2;
        a.err = err;
        e = m.r.bits == 8 ? launch_answer<8>(a, st) : launch_answer<4>(a, st);
    }
    return e;
}

}  // namespace vdb
