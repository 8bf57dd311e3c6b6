// Quantised speaker registry: embeddings are quantised as they are written and read back
// as unit vectors; queries are scored against the stored rows, or turned into a posterior
// over the enrolled speakers without storing the scores. No reference counterpart exists
// (the reference keeps no registry); format and semantics: vdb_ops.h.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <mutex>
#include <string>
#include <type_traits>

#include "registry.cuh"

namespace vdb {
namespace {

// ---------------------------------------------------------------------------
// clear, write, read
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
registry_clear_kernel(float* scale, int* owner, int capacity, const int* __restrict__ slots,
                      int first, int n) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;  // (n up to 2^31 - 1)
    if (i >= (unsigned)n) return;
    const int s = slots ? slots[i] : first + (int)i;
    if (s < 0 || s >= capacity) return;
    scale[s] = __int_as_float(0x7FC00000);
    if (!slots) owner[s] = -1;
}

// The last row of each slot: owner[slot] = the highest row index that names it. The write
// kernel's winner puts the -1 back, so the array is ready for the next call.
__global__ void __launch_bounds__(256)
registry_claim_kernel(int* owner, int capacity, const int* __restrict__ slots, int n) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= (unsigned)n) return;
    const int s = slots[i];
    if (s >= 0 && s < capacity) atomicMax(owner + s, (int)i);
}

// Eight consecutive elements of a row as they are in memory (VEC: 16-byte aligned, and the row
// ends at a multiple of eight) or as f32, 0 from `left` on.
template <typename T, bool VEC>
struct Eight {
    static constexpr int kWords = VEC && sizeof(T) == 2 ? 1 : 2;
    uint4 w[kWords];

    __device__ __forceinline__ void load(const T* p, int left) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (VEC) {
            if (left > 0)
#pragma unroll
                for (int i = 0; i < kWords; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        } else {
            float v[8];
            emb8(p, sizeof(T) == 4 ? kF32 : std::is_same_v<T, __half> ? kF16 : kBF16, 0, left, v);
            w[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                              __float_as_uint(v[3]));
            w[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]),
                              __float_as_uint(v[7]));
        }
    }
    __device__ __forceinline__ void pairs(f2 (&v)[4]) const {
        if constexpr (kWords == 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[2 * i] = pack2(__uint_as_float(w[i].x), __uint_as_float(w[i].y));
                v[2 * i + 1] = pack2(__uint_as_float(w[i].z), __uint_as_float(w[i].w));
            }
        } else {
            const uint32_t x[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (std::is_same_v<T, __half>) {
                    __half2 h;
                    memcpy(&h, &x[i], 4);
                    const float2 f = __half22float2(h);
                    v[i] = pack2(f.x, f.y);
                } else {  // bf16 is the upper half of an f32
                    v[i] = pack2(__uint_as_float(x[i] << 16), __uint_as_float(x[i] & 0xFFFF0000u));
                }
            }
        }
    }
};

// A warp takes up to write_rows rows, all loaded before the first is used (one row a warp
// keeps too few bytes on their way), eight consecutive dimensions per lane and NIT steps of
// 256. A quotient x f (f = 127 / max or 889 / (max s) in f32) is rounded by one fused
// multiply-add onto 1.5 2^23 + the code's offset, whose low bits are the code, two at a time.
// One that lands within the f32 error of a half (8 bits: 2e-5, f errs by 127 2^-24 = 8e-6; 4
// bits: 1e-5, 7 (2^-22 + 2^-24) = 2e-6) sends its lane's eight through f64 quotients, which
// are exact enough to tell the sides apart (of rows of 256 dimensions one in 100 with 8 bits, one
// in 200 with 4); the group scale's whole-number
// border is treated alike. HBM bound (4 dim bytes in, dim bits / 8 out) as long as a row takes
// few instructions: the rows' f64 scales are therefore taken side by side at the end, one a
// lane. 100,000 f32 rows of 256 dimensions: 26 us to 8 bits (4.9 TB/s), 32 us to 4 (3.7 TB/s).
constexpr int write_rows(int nit, int words) { return nit * words >= 4 ? 1 : 4 / (nit * words); }

template <typename T, int BITS, int NIT, bool VEC>
__global__ void __launch_bounds__(256)
registry_write_kernel(const T* __restrict__ x, long long ldx, const int* __restrict__ slots,
                      int first, int n, int capacity, int dim, int dim_pad, int gpitch,
                      long long row_bytes, uint8_t* codes, uint8_t* group, float* scale,
                      int* owner, int per_warp) {
    const int lane = threadIdx.x & 31;
    const long long i0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * per_warp;
    if (i0 >= n) return;
    const int rows = (int)min((long long)per_warp, n - i0);
    constexpr float kMagic = 12582912.0f;
    constexpr int kOffset = BITS == 8 ? 128 : 8;
    constexpr int kRows = write_rows(NIT, Eight<T, VEC>::kWords);
    Eight<T, VEC> all[kRows][NIT];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const T* row = x + (i0 + (r < rows ? r : 0)) * ldx + lane * 8;
#pragma unroll
        for (int it = 0; it < NIT; ++it)
            all[r][it].load(row + it * 256, dim - lane * 8 - it * 256);
    }
    // lane r: slot of row r (-1: skipped), its sum of squares (-1: an infinity or a NaN)
    int slot = -1, square = 0;
    if (lane < rows) {
        slot = slots ? slots[i0 + lane] : first + (int)i0 + lane;
        if (slot < 0 || slot >= capacity) slot = -1;
        if (owner && slot >= 0) {
            if (owner[slot] == (int)i0 + lane)
                owner[slot] = -1;
            else
                slot = -1;
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (r >= rows) break;
        const int at = __shfl_sync(0xffffffffu, slot, r);
        if (at < 0) continue;
        f2 v[NIT][4];
        float gm[NIT], most = 0.0f;
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
            all[r][it].pairs(v[it]);
            gm[it] = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float a, b;
                unpack2(v[it][j], a, b);
                gm[it] = fmaxf(gm[it], fmaxf(fabsf(a), fabsf(b)));
            }
            most = fmaxf(most, gm[it]);
        }
        // (a NaN shows in the sum of squares, an infinity here)
        const float top =
            __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
        // outside this range a quotient's f32 factor could leave f32's normal range
        const bool fast = top > 1e-30f && top < 1e30f;
        const float inv = fast ? 127.0f / top : 0.0f;
        bool bad = !(top <= FLT_MAX);
        int sum = 0;
        uint8_t* out = codes + at * row_bytes + lane * BITS;
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
            float f = inv;
            int si = 1;
            if constexpr (BITS == 4) {
                float g = fmaxf(gm[it], __shfl_xor_sync(0xffffffffu, gm[it], 1));
                g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
                const float y = g * inv;
                float s = g == top && g > 0.0f ? 127.0f : ceilf(y);
                const bool near = g > 0.0f && g != top && (!fast || fabsf(y - rintf(y)) < 1e-4f);
                if (__any_sync(0xffffffffu, near) && near)
                    s = (float)ceil(127.0 * (double)g / (double)top);
                f = fast && s > 0.0f ? __fdividef(889.0f, top * s) : 0.0f;
                si = (int)s;
            }
            // u = -w, and how far x f is from w
            const f2 ff = pack2(f, f), magic = pack2(kMagic + kOffset, kMagic + kOffset);
            const f2 minus = pack2(-1.0f, -1.0f);
            f2 u[4], sq = 0ull;
            float far = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] = fma2(fma2(v[it][j], ff, magic), minus, magic);
                sq = fma2(u[j], u[j], sq);
                float a, b;
                unpack2(fma2(v[it][j], ff, u[j]), a, b);
                far = fmaxf(far, fmaxf(fabsf(a), fabsf(b)));
            }
            const bool near =
                (!fast && si != 0 && top > 0.0f) || far > (BITS == 8 ? 0.49998f : 0.49999f);
            if (__any_sync(0xffffffffu, near) && near) {
                const double den = BITS == 8 ? (double)top : (double)top * (double)si;
                sq = 0ull;
#pragma unroll 1
                for (int j = 0; j < 4; ++j) {
                    f2 vj = v[it][0];
#pragma unroll
                    for (int i = 1; i < 4; ++i) vj = j == i ? v[it][i] : vj;
                    float a, b;
                    unpack2(vj, a, b);
                    a = (float)rint((BITS == 8 ? -127.0 : -889.0) * (double)a / den);
                    b = (float)rint((BITS == 8 ? -127.0 : -889.0) * (double)b / den);
                    const f2 uj = pack2(a, b);
                    sq = fma2(uj, uj, sq);
#pragma unroll
                    for (int i = 0; i < 4; ++i) u[i] = j == i ? uj : u[i];
                }
            }
            float sa, sb;
            unpack2(sq, sa, sb);
            sa += sb;  // whole numbers below 2^24: exact
            bad |= sa != sa;
            sum += (int)sa * si * si;
            if constexpr (BITS == 8) {
                uint32_t lo[4], word[2];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f2 q = fma2(u[j], minus, magic);  // w + 128 in the low byte
                    lo[j] = __byte_perm((uint32_t)q, (uint32_t)(q >> 32), 0x0040);
                }
                word[0] = __byte_perm(lo[0], lo[1], 0x5410);
                word[1] = __byte_perm(lo[2], lo[3], 0x5410);
                if (it * 256 + lane * 8 < dim_pad)
                    *reinterpret_cast<uint2*>(out + it * 256) = make_uint2(word[0], word[1]);
            } else {
                // four nibbles (dimensions 0, 2, 4, 6 and 1, 3, 5, 7) as one number below 2^16,
                // exact in f32, read from its low bits
                f2 n = fma2(u[0], minus, pack2(kMagic + 8 * 4369, kMagic + 8 * 4369));
                n = fma2(u[1], pack2(-16.0f, -16.0f), n);
                n = fma2(u[2], pack2(-256.0f, -256.0f), n);
                n = fma2(u[3], pack2(-4096.0f, -4096.0f), n);
                if (it * 256 + lane * 8 < dim_pad) {
                    *reinterpret_cast<uint32_t*>(out + it * 128) =
                        __byte_perm((uint32_t)n, (uint32_t)(n >> 32), 0x5410);
                    if ((lane & 3) == 0)
                        group[(long long)at * gpitch + it * 8 + lane / 4] = (uint8_t)si;
                }
            }
        }
        if (__any_sync(0xffffffffu, bad)) {
            // nothing of the row is kept: zeros, and the slot is empty
            sum = 0;
#pragma unroll
            for (int it = 0; it < NIT; ++it) {
                if (it * 256 + lane * 8 >= dim_pad) continue;
                if constexpr (BITS == 8) {
                    *reinterpret_cast<uint2*>(out + it * 256) = make_uint2(0x80808080u, 0x80808080u);
                } else {
                    *reinterpret_cast<uint32_t*>(out + it * 128) = 0x88888888u;
                    if ((lane & 3) == 0) group[(long long)at * gpitch + it * 8 + lane / 4] = 0;
                }
            }
            bad = true;
        }
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == r) square = bad ? -1 : sum;
    }
    if (slot >= 0)
        scale[slot] = square < 0 ? __int_as_float(0x7FC00000)
                                 : (square > 0 ? (float)rsqrt((double)square) : 0.0f);
}

__device__ __forceinline__ uint16_t bits16(__half v) { return __half_as_ushort(v); }
__device__ __forceinline__ uint16_t bits16(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// Four values to a row, `left` of them inside it.
__device__ __forceinline__ void store4(float* p, int left, bool vec, const float (&v)[4]) {
    if (vec && left >= 4) {
        __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < left) p[j] = v[j];
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int left, bool vec, const float (&v)[4]) {
    T h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) from_f32(v[j], h[j]);
    if (vec && left >= 4) {
        __stcs(reinterpret_cast<uint2*>(p),
               make_uint2((uint32_t)bits16(h[0]) | (uint32_t)bits16(h[1]) << 16,
                          (uint32_t)bits16(h[2]) | (uint32_t)bits16(h[3]) << 16));
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < left) p[j] = h[j];
}

// One warp per row, four consecutive dimensions per lane and step, so that a store
// instruction writes whole 32-byte sectors. HBM bound: dim bits / 8 bytes in, 4 (2) dim out;
// 100,000 4-bit rows of 256 dimensions to f32: 21 us (5.4 TB/s).
template <typename T, int BITS>
__global__ void __launch_bounds__(256)
registry_read_kernel(RegDev r, int capacity, const int* __restrict__ slots, int first, int n,
                     T* __restrict__ out, long long ldo, bool vec) {
    const unsigned i = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= (unsigned)n) return;
    const int slot = slots ? slots[i] : first + (int)i;
    const bool inside = slot >= 0 && slot < capacity;
    // outside: row 0's codes times NaN
    const long long at = inside ? slot : 0;
    const float scale = inside ? r.scale[at] : __int_as_float(0x7FC00000);
    const uint8_t* codes = r.codes + at * r.row_bytes;
    const uint8_t* group = r.group + at * r.gpitch;
    T* row = out + (long long)i * ldo;
#pragma unroll 4
    for (int d0 = lane * 4; d0 < r.dim; d0 += 128) {
        // a code in the low bits of 2^23 is 2^23 + code; the offset comes off exactly
        float v[4];
        if constexpr (BITS == 8) {
            const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + d0);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = (__uint_as_float(__byte_perm(c, 0x4B000000u, 0x7440 + j)) - 8388736.0f) * scale;
        } else {
            // dimensions 0, 1, 2, 3 of the word's eight are nibbles 0, 4, 1, 5; 4 to 7 sit
            // eight bits higher
            uint32_t c = *reinterpret_cast<const uint32_t*>(codes + (d0 & ~7) / 2);
            c >>= (d0 & 4) * 2;
            const float s = (float)group[d0 >> 5];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t nib = (c >> ((j & 1) * 16 + (j >> 1) * 4)) & 15u;
                v[j] = (__uint_as_float(0x4B000000u | nib) - 8388616.0f) * s * scale;
            }
        }
        store4(row + d0, r.dim - d0, vec, v);
    }
}

// ---------------------------------------------------------------------------
// a few queries: warp-level matrix products straight from the stored codes
// ---------------------------------------------------------------------------
constexpr int kFewThreads = 256;
constexpr int kFewMaxSeg = 4096;  // rows a block scores at most: a part of kPart a warp

struct FewArgs {
    RegDev r;
    int n_rows;
    const void* q;
    int q_type;
    long long ldq;
    int n_q;
    int rows_per, n_slices;  // rows per block (a multiple of 16), blocks per query group
    int pitch;               // scores' shared-memory pitch
    float* out;              // scores
    long long ldo;
    float s2;                // temperature * log2(e)
    int L;                   // candidates wanted
    RegParts parts;
};

// Bytes of shared memory that a block's queries take.
__host__ __device__ inline size_t few_query_bytes(int nt, int dim_pad) {
    // one 4-bit query: per 128 dimensions four operand fragments a lane and a pair of
    // starting values a group; the query's unit
    if (nt == 0) {
        const int n_b = (dim_pad + 127) / 128;
        return (size_t)n_b * (4 * 32 * 16 + 4 * 8) + 16;
    }
    return (size_t)8 * nt * (dim_pad + 8) * 2;
}

// 256 dimensions (two blocks of 128) of rows g + 8 i for the one-query product over 4-bit
// codes: lane t holds all of group t of each block (32 dimensions, 16 bytes) and the eight
// group scales.
struct OneFrag {
    uint4 x[2][4];
    uint2 s[4];
};

// A block holds 4 NT queries as B operands (column pairs: high and low part of one query's
// unit vector) in shared memory and scores rows_per rows, 16 per warp-level m16n8k16
// product, widening the codes in registers. Lane (g, t) loads 16 consecutive dimensions
// 16 t .. 16 t + 15 of rows g and g + 8 per 64: the products' k index is a permutation of
// the dimensions, the same for both operands. It ends up with the scores of query t.
//
// NT = 0 is one query over 4-bit codes, where widening would cost more than the bytes: the
// product's columns are (group t', part) pairs instead, the query masked to the 32
// dimensions (16 bytes) that lane t' holds of each 128, so that an accumulator is one
// group's product with the bare codes and the group's scale multiplies once per 128
// dimensions; a warp takes 32 rows a step. The query is in fixed point (split_query_fixed), so
// that a group's products and sums are whole numbers below 2^24 and exact. A nibble in bits 0-3
// or 4-7 of a zero f16 is the code's value times 2^-24 or 2^-20 (a subnormal, exact), one
// mask per two codes; the operand of the latter is a sixteenth of the query, and the
// offset 8 of the stored codes is subtracted by starting at -8 times the query's sum.
//
// The next 256 dimensions are loaded before the current ones are used (NT <= 2), or right
// after (more queries: the registers are short, and the products of two blocks an SM cover
// more of the loads).
//
// Bound by HBM with one query: the scores of 2,000,003 4-bit rows of 256 dimensions take 53 us
// (5.5 TB/s with the output), 1,000,000 8-bit rows 40 us (6.5 TB/s). With more queries by what
// comes before and after the rows: 12 queries' posterior over 100,000 8-bit rows is 15 us, 2.4
// of it the queries' unit vectors, 5.3 the rows (4.9 TB/s) and 4.6 the selection.
template <int BITS, int NT, bool POST>
__global__ void __launch_bounds__(kFewThreads, 2)
registry_few_kernel(const __grid_constant__ FewArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int kQueries = NT ? 4 * NT : 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int slice = blockIdx.x % p.n_slices, q0 = blockIdx.x / p.n_slices * kQueries;
    const int nq = min(kQueries, p.n_q - q0);
    const int qpitch = p.r.dim_pad + 8;  // halfs
    __half* qs = reinterpret_cast<__half*>(smem);
    float* sc = reinterpret_cast<float*>(smem + few_query_bytes(NT, p.r.dim_pad));
    if constexpr (POST) pdl_launch_dependents();
    const int r0 = slice * p.rows_per;
    const int rows = min(p.rows_per, p.n_rows - r0);
    constexpr int kWarps = kFewThreads / 32;
    const uint64_t policy = code_policy(p.r.once);
    if constexpr (NT == 0) {
        const int n_b = (p.r.dim_pad + 127) / 128, n_groups = p.r.dim_pad / 32;
        uint4* frag = reinterpret_cast<uint4*>(smem);                 // [n_b][4][32 lanes]
        float2* start = reinterpret_cast<float2*>(frag + n_b * 128);  // [n_b * 4 groups], unit
        const uint8_t* codes = p.r.codes + r0 * p.r.row_bytes;
        const uint8_t* group = p.r.group + (long long)r0 * p.r.gpitch;
        const uint32_t rb = (uint32_t)p.r.row_bytes, gp = (uint32_t)p.r.gpitch;
        OneFrag f[2];
        float scale = 0.0f;  // of the row whose score this lane keeps: g + 8 t of the 32
        auto fetch = [&](OneFrag& x, int pair, int b0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t r = (uint32_t)min(pair * 32 + g + 8 * i, rows - 1);
                const uint32_t off = r * rb + 16u * t + 64u * b0;
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if ((b0 + u) * 4 + t < n_groups)
                        x.x[u][i] = load_codes16(codes + (off + 64u * u), policy);
                x.s[i] = __ldg(reinterpret_cast<const uint2*>(group + (r * gp + 4u * b0)));
            }
            if (b0 == 0) scale = __ldg(p.r.scale + r0 + min(pair * 32 + g + 8 * t, rows - 1));
        };
        int pair = warp, b0 = 0;
        if (pair * 32 < rows) fetch(f[0], pair, 0);
        // fragment m of lane (g, t): the query's part g & 1 where g / 2 is the lane's own group,
        // 0 elsewhere; a sixteenth of it where the codes sit in bits 4-7
        for (int i = threadIdx.x; i < n_b * 128; i += kFewThreads)
            if (((i & 31) >> 3) != (i & 3)) frag[i] = make_uint4(0u, 0u, 0u, 0u);
        if (warp == 0) {
            const float unit = split_query_fixed(
                p.q, p.q_type, (long long)q0 * p.ldq, p.r.dim, n_b * 128,
                [&](int d0, const uint32_t(&h)[4], const uint32_t(&l)[4]) {
                    // eight dimensions: one fragment; four lanes: one group
                    const int grp = d0 >> 5, m = (d0 >> 3) & 3, at = grp & 3;
                    uint4* f = frag + (d0 >> 7) * 128 + m * 32 + 8 * at + at;
                    const uint32_t sixteenth = 0x2C002C00u, zero = 0x80008000u;
                    f[0] = make_uint4(h[0], h2_fma(h[1], sixteenth, zero), h[2],
                                      h2_fma(h[3], sixteenth, zero));
                    f[4] = make_uint4(l[0], h2_fma(l[1], sixteenth, zero), l[2],
                                      h2_fma(l[3], sixteenth, zero));
                    // -8 times the parts' sums, in the nibbles' unit 2^-24
                    float2 s = make_float2(h2_sum(h[0]) + h2_sum(h[1]),
                                           h2_sum(l[0]) + h2_sum(l[1]));
                    s.x += h2_sum(h[2]) + h2_sum(h[3]);
                    s.y += h2_sum(l[2]) + h2_sum(l[3]);
#pragma unroll
                    for (int o = 1; o <= 2; o <<= 1) {
                        const unsigned four = 0xFu << (lane & 28);
                        s.x += __shfl_xor_sync(four, s.x, o);
                        s.y += __shfl_xor_sync(four, s.y, o);
                    }
                    if ((lane & 3) == 0)
                        start[grp] = make_float2(s.x * (-8.0f / 16777216.0f),
                                                 s.y * (-8.0f / 16777216.0f));
                });
            if (lane == 0) start[n_b * 4].x = unit * 16777216.0f;
        }
        __syncthreads();
        const float unit = start[n_b * 4].x;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        // one step of 256 dimensions with `cur`, the next one's data on its way to `next`;
        // false after the warp's last rows
        auto step = [&](const OneFrag& cur, OneFrag& next) {
            const bool last = b0 + 2 >= n_b;
            const int npair = last ? pair + kWarps : pair, nb0 = last ? 0 : b0 + 2;
            const bool more = npair * 32 < rows;
            const float cs = scale;
            if (more) fetch(next, npair, nb0);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (b0 + u >= n_b) break;
                const float2 s0 = start[(b0 + u) * 4 + t];
                float acc[2][4] = {{s0.x, s0.y, s0.x, s0.y}, {s0.x, s0.y, s0.x, s0.y}};
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const uint4 b = frag[(b0 + u) * 128 + m * 32 + lane];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 &xa = cur.x[u][2 * h], &xb = cur.x[u][2 * h + 1];
                        const uint32_t wa = m == 0 ? xa.x : m == 1 ? xa.y : m == 2 ? xa.z : xa.w;
                        const uint32_t wb = m == 0 ? xb.x : m == 1 ? xb.y : m == 2 ? xb.z : xb.w;
                        const uint32_t a8 = wa >> 8, b8 = wb >> 8;
                        mma_16816(acc[h], wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u,
                                  wb & 0x00F000F0u, b.x, b.y);
                        mma_16816(acc[h], a8 & 0x000F000Fu, b8 & 0x000F000Fu, a8 & 0x00F000F0u,
                                  b8 & 0x00F000F0u, b.z, b.w);
                    }
                }
                // a lane past the row's groups holds nothing: its scale is 0
                const bool in = (b0 + u) * 4 + t < n_groups;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t sg = u ? cur.s[i].y : cur.s[i].x;
                    const float f = in ? (float)__byte_perm(sg, 0u, 0x4440u + t) : 0.0f;
                    const float* c = acc[i >> 1] + 2 * (i & 1);
                    v[i] = fmaf(fmaf(c[0], 4096.0f, c[1]), f, v[i]);
                }
            }
            if (last) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // over the four groups of each block
                    v[i] += __shfl_xor_sync(0xffffffffu, v[i], 1);
                    v[i] += __shfl_xor_sync(0xffffffffu, v[i], 2);
                }
                const float mine = t == 0 ? v[0] : t == 1 ? v[1] : t == 2 ? v[2] : v[3];
                const float score = cs == cs ? mine * (unit * cs) : -INFINITY;
                const int at = pair * 32 + g + 8 * t;
                if (at < rows) {
                    if constexpr (POST)
                        sc[at] = score;
                    else
                        p.out[(long long)q0 * p.ldo + r0 + at] = score;
                }
                v[0] = v[1] = v[2] = v[3] = 0.0f;
            }
            pair = npair;
            b0 = nb0;
            return more;
        };
        if (pair * 32 < rows)
            while (step(f[0], f[1]) && step(f[1], f[0])) {
            }
    } else {
        constexpr bool kAhead = NT <= 2;
        const int n_chunks = p.r.dim_pad / 64;
        int tile = warp, c0 = 0;
        long long ga = r0 + min(tile * 16 + g, rows - 1), gb = r0 + min(tile * 16 + g + 8, rows - 1);
        RowFrag<BITS> cur;
        if (tile * 16 < rows) cur.load(p.r, ga, gb, 0, n_chunks, t, policy);
#pragma unroll 2
        for (int j = warp; j < 4 * NT; j += kWarps) {
            __half* hi = qs + (size_t)((j >> 2) * 8 + (j & 3) * 2) * qpitch;
            split_query(p.q, p.q_type, (long long)(q0 + j) * p.ldq, p.r.dim, p.r.dim_pad, j < nq,
                        StoreParts{hi, hi + qpitch});
        }
        __syncthreads();
        float acc[NT ? NT : 1][4] = {};
        float sa = p.r.scale[ga], sb = p.r.scale[gb];
        while (tile * 16 < rows) {
            int ntile = tile, nc0 = c0 + 4;
            if (nc0 >= n_chunks) {
                nc0 = 0;
                ntile += kWarps;
            }
            long long na = ga, nb = gb;
            if (ntile != tile) {
                na = r0 + min(ntile * 16 + g, rows - 1);
                nb = r0 + min(ntile * 16 + g + 8, rows - 1);
            }
            RowFrag<BITS> next;
            if constexpr (kAhead) {
                if (ntile * 16 < rows) next.load(p.r, na, nb, nc0, n_chunks, t, policy);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (c0 + u >= n_chunks) break;
                uint32_t fa[8], fb[8];
                cur.widen(u, t, fa, fb);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const uint4* qb = reinterpret_cast<const uint4*>(
                        qs + (size_t)(i * 8 + g) * qpitch + (c0 + u) * 64 + 16 * t);
                    const uint4 b0 = qb[0], b1 = qb[1];
                    mma_16816(acc[i], fa[0], fb[0], fa[1], fb[1], b0.x, b0.y);
                    mma_16816(acc[i], fa[2], fb[2], fa[3], fb[3], b0.z, b0.w);
                    mma_16816(acc[i], fa[4], fb[4], fa[5], fb[5], b1.x, b1.y);
                    mma_16816(acc[i], fa[6], fb[6], fa[7], fb[7], b1.z, b1.w);
                }
            }
            if (!kAhead && ntile * 16 < rows) cur.load(p.r, na, nb, nc0, n_chunks, t, policy);
            if (ntile != tile) {
                const int at = tile * 16 + g;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const int j = i * 4 + t;
                    const float va =
                        sa == sa ? (acc[i][0] + acc[i][1]) * (sa * (1.0f / kQScale)) : -INFINITY;
                    const float vb =
                        sb == sb ? (acc[i][2] + acc[i][3]) * (sb * (1.0f / kQScale)) : -INFINITY;
                    acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
                    if (j >= nq) continue;
                    if constexpr (POST) {
                        if (at < rows) sc[j * p.pitch + at] = va;
                        if (at + 8 < rows) sc[j * p.pitch + at + 8] = vb;
                    } else {
                        float* o = p.out + (long long)(q0 + j) * p.ldo + r0;
                        if (at < rows) o[at] = va;
                        if (at + 8 < rows) o[at + 8] = vb;
                    }
                }
                if (ntile * 16 < rows) {
                    sa = p.r.scale[na];
                    sb = p.r.scale[nb];
                }
            }
            tile = ntile;
            c0 = nc0;
            ga = na;
            gb = nb;
            if constexpr (kAhead) cur = next;
        }
    }
    if constexpr (POST) {
        __syncthreads();
        // a partial per kPart rows (the last block's may be empty)
        const int per = (p.rows_per + kPart - 1) / kPart, cap = p.parts.cap;
        for (int task = warp; task < nq * per; task += kWarps) {
            const int j = task / per, part = task - j * per;
            const long long at = ((long long)slice * per + part) * p.n_q + q0 + j;
            const auto select = [&](auto slots) {
                return warp_select<decltype(slots)::value>(
                    sc + j * p.pitch + part * kPart, nullptr, r0 + part * kPart,
                    max(0, min(kPart, rows - part * kPart)), p.L, cap, p.s2,
                    p.parts.score + at * cap, p.parts.slot + at * cap);
            };
            const RegPart st = p.rows_per <= 256 ? select(std::integral_constant<int, 8>())
                                                 : select(std::integral_constant<int, kPart / 32>());
            if (lane == 0) p.parts.stat[at] = st;
        }
    }
}

// ---------------------------------------------------------------------------
// merging the partials of a query, exact rescoring, the posterior
// ---------------------------------------------------------------------------
constexpr int kMergeThreads = 256;
constexpr int kMergeSome = 160;  // candidates a block ranks at most
// Up to as many candidates wanted 1024 are held in shared memory (21 KB), otherwise 2816 (36
// KB): the blocks have to fit beside the few-query kernel's, or they start late (12 queries x
// 100,000 rows, k = 5: 21.8 us, with the larger ones 23.1, or 22.4 with more shared memory set
// aside).
constexpr int kMergeSmallL = 32;

// One block per query: the best L candidates over the partials (by their f32 scores), each
// and the label's slot rescored in f64, and the softmax of all of it around the exact top
// score M: with E the sum of exp(z - M) over everything but the top, lse = M + log1p(E) and
// log p(top) = -log1p(E). Sums run in an order fixed by the sizes alone. The block's queries
// are staged while the scores are still being computed; after them its time is a chain of
// latencies (partials, the few lists that reach the bound, the candidates' rows, f64 tail).
// CAND: candidates held in shared memory. 7 to 8 us after the scores for k = 5, 12 for k = 20,
// 20 for k = 64.
template <int CAND>
__global__ void __launch_bounds__(kMergeThreads)
registry_merge_kernel(const __grid_constant__ MergeArgs p) {
    __shared__ __align__(16) double qv[kRegMaxDim];
    __shared__ float head[kMergeThreads];
    __shared__ float cs[CAND];
    __shared__ int ci[CAND];
    __shared__ float few_s[kMergeSome];
    __shared__ int few_i[kMergeSome];
    __shared__ int hot[kMergeThreads];
    __shared__ float bs[kRegMaxK + kRegExtra];  // candidates by rank
    __shared__ int bi[kRegMaxK + kRegExtra];
    __shared__ double ex[kRegMaxK + kRegExtra + 1];
    __shared__ int rank[kRegMaxK + kRegExtra];
    __shared__ double s_qq;
    __shared__ float red[2][kMergeThreads / 32];
    __shared__ int s_cnt, s_hot, s_ties, s_few;
    __shared__ uint2 s_round[2][kMergeThreads / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int qi = blockIdx.x;
    const int L = p.L, cap = p.parts.cap, n_part = p.parts.n_part;
    const float s2 = p.temperature * 1.4426950408889634f;
    if (warp == 0) {
        const double s = stage_query(p, qi, qv);
        if (lane == 0) s_qq = s;
    }
    const int label = label_of(p, qi);
    if (tid == 0) s_cnt = 0, s_hot = 0, s_ties = 0, s_few = 0;
    pdl_wait();

    // each thread's parts, its sums relative to their best score hm: everything but one score
    // equal to hm (parts that reach hm leave theirs out, all of them but one are put back)
    const RegPart* stat = p.parts.stat + qi;
    float hm = -INFINITY, e0 = 0.0f, e1 = 0.0f;
    const auto take = [&](const RegPart& o) {
        if (o.ref == -INFINITY) return;
        if (o.ref > hm) {
            // what there was, hm's score included, against the new best one
            const float d = (hm - o.ref) * s2, f = exp2f(d);
            const bool some = hm > -INFINITY;
            const float s = some ? e0 + 1.0f : 0.0f;
            e1 = o.e1 + (some ? f * (e1 + s * d) : 0.0f);
            e0 = o.e0 + f * s;
            hm = o.ref;
        } else {
            const float d = (o.ref - hm) * s2, f = exp2f(d), s = o.e0 + 1.0f;
            e0 += f * s;
            e1 += f * (o.e1 + s * d);
        }
    };
    for (int i0 = tid; i0 < n_part; i0 += 4 * kMergeThreads) {
        RegPart o[4];  // four loads on their way
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * kMergeThreads;
            o[u].ref = -INFINITY;
            if (i < n_part) o[u] = stat[(long long)i * p.n_q];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) take(o[u]);
    }
    head[tid] = hm;
    __syncthreads();
    // every warp: the best score, and a bound that the L-th best reaches
    uint32_t key[kMergeThreads / 32], ckey = 0;
#pragma unroll
    for (int i = 0; i < kMergeThreads / 32; ++i) {
        const float h = head[lane + 32 * i];
        key[i] = h > -INFINITY ? key_of(h) : 0u;
        ckey = max(ckey, key[i]);
    }
    const uint32_t top_key = __reduce_max_sync(0xffffffffu, ckey);
    // (of the 32 lanes' maxima where that is enough; fewer parts than that give none)
    const uint32_t bound = n_part < L ? 1u
                           : L <= 32  ? max(lth_lane_key(ckey, L), 1u)
                                      : max(lth_key<kMergeThreads / 32>(key, L), 1u);
    const float ref = top_key == 0 ? -INFINITY : from_key(top_key);
    for (int i = tid; i < n_part; i += kMergeThreads) {
        const float r = stat[(long long)i * p.n_q].ref;
        if (r > -INFINITY && key_of(r) >= bound) {
            const int pos = atomicAdd(&s_hot, 1);
            if (pos < kMergeThreads) hot[pos] = i;
        }
    }
    if (hm > -INFINITY) {
        // relative to ref, everything but one score equal to it
        const bool at_top = hm == ref;
        if (at_top) atomicAdd(&s_ties, 1);
        const float d = (hm - ref) * s2, f = exp2f(d), s = e0 + (at_top ? 0.0f : 1.0f);
        e1 = f * (e1 + s * d);
        e0 = f * s;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        e0 += __shfl_xor_sync(0xffffffffu, e0, o);
        e1 += __shfl_xor_sync(0xffffffffu, e1, o);
    }
    if (lane == 0) red[0][warp] = e0, red[1][warp] = e1;
    __syncthreads();
    const int n_hot = s_hot;
    auto entry = [&](int part, int j, float& s, int& i) {
        const long long o = ((long long)part * p.n_q + qi) * cap + j;
        s = p.parts.score[o];
        i = p.parts.slot[o];
    };
    auto collect = [&](uint32_t least, int n, bool all) {
        for (int e0 = 0; e0 < n * cap; e0 += 4 * kMergeThreads) {
            float s[4];
            int i[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int e = e0 + u * kMergeThreads + tid, part = e / cap;
                i[u] = -1;
                if (e < n * cap) entry(all ? part : hot[part], e - part * cap, s[u], i[u]);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool in = i[u] >= 0 && key_of(s[u]) >= least;
                const unsigned m = __ballot_sync(0xffffffffu, in);
                int pos = 0;
                if (lane == 0 && m != 0) pos = atomicAdd(&s_cnt, __popc(m));
                pos = __shfl_sync(0xffffffffu, pos, 0) + __popc(m & ((1u << lane) - 1u));
                if (in && pos < CAND) cs[pos] = s[u], ci[pos] = i[u];
            }
        }
        __syncthreads();
        return s_cnt;
    };
    int cnt = CAND + 1;
    if (n_hot <= kMergeThreads) cnt = collect(bound, n_hot, false);
    if (cnt > CAND) {
        // many lists or entries reach the bound: bisection in the scores for one that L to
        // CAND reach (all of them above lo, at least L above -FLT_MAX)
        float lo = from_key(bound), hi = ref;
        if (!(lo > -FLT_MAX)) lo = -fabsf(ref) - 2.1f;  // below every cosine
        while (true) {
            const float mid = 0.5f * lo + 0.5f * hi;
            const bool last = !(mid > lo && mid < hi);
            const float least = last ? lo : mid;
            int c = 0;
            for (int e = tid; e < n_part * cap; e += kMergeThreads) {
                float s;
                int i;
                entry(e / cap, e % cap, s, i);
                c += i >= 0 && s >= least ? 1 : 0;
            }
            __syncthreads();  // the previous round's count has been read
            if (tid == 0) s_cnt = 0;
            __syncthreads();
            c = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0) atomicAdd(&s_cnt, c);
            __syncthreads();
            c = s_cnt;
            if (last || (c >= L && c <= CAND)) {
                lo = least;
                break;
            }
            if (c >= L)
                lo = mid;
            else
                hi = mid;
        }
        __syncthreads();
        if (tid == 0) s_cnt = 0;
        __syncthreads();
        cnt = collect(key_of(lo), n_part, true);
    }
    const float* list_s = cs;
    const int* list_i = ci;
    if (cnt > kMergeSome && cnt <= CAND) {
        // the same among the candidates held, for a bound that L to kMergeSome reach; where
        // equal scores leave none, bisection in their slots goes on from there
        constexpr int kMine = CAND / kMergeThreads;
        float a[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int e = tid + i * kMergeThreads;
            a[i] = e < cnt ? cs[e] : -INFINITY;
        }
        int round = 0;
        // four counts at once, 16 bits each, over the block
        const auto total = [&](const int(&c)[4], int (&sum)[4]) {
            const uint32_t w0 = __reduce_add_sync(0xffffffffu, (uint32_t)(c[0] | c[1] << 16));
            const uint32_t w1 = __reduce_add_sync(0xffffffffu, (uint32_t)(c[2] | c[3] << 16));
            uint2* at = s_round[round & 1];
            round ^= 1;
            if (lane == 0) at[warp] = make_uint2(w0, w1);
            __syncthreads();
            uint32_t v0 = 0, v1 = 0;
#pragma unroll
            for (int w = 0; w < kMergeThreads / 32; ++w) v0 += at[w].x, v1 += at[w].y;
            sum[0] = (int)(v0 & 0xFFFFu), sum[1] = (int)(v0 >> 16);
            sum[2] = (int)(v1 & 0xFFFFu), sum[3] = (int)(v1 >> 16);
        };
        const auto fits = [&](int c) { return c >= L && c <= kMergeSome; };
        float lo = -fabsf(ref) - 2.1f, hi = ref, least = hi;
        int upto = INT_MAX, c = 0;
        while (true) {
            // four bounds between lo and hi; hi where there is no number for one
            float t[4], nlo = lo, nhi = hi;
            int part[4], sum[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                t[u] = lo + (hi - lo) * (0.2f * (float)(u + 1));
                if (!(t[u] > lo && t[u] < hi)) t[u] = hi;
                part[u] = 0;
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    if (i * kMergeThreads >= cnt) break;
                    part[u] += a[i] >= t[u] ? 1 : 0;
                }
            }
            total(part, sum);
            bool found = false;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (fits(sum[u])) {
                    found = true;
                    least = t[u];
                    c = sum[u];
                } else if (t[u] < hi) {
                    if (sum[u] >= L)
                        nlo = fmaxf(nlo, t[u]);
                    else
                        nhi = fminf(nhi, t[u]);
                }
            }
            if (found) break;
            if (nlo == lo && nhi == hi) {
                // none between: equal scores, at hi or (fewer than L reach hi) at lo
                least = sum[0] < L ? lo : hi;
                int below = -1, above = p.n_rows - 1;
                do {
                    upto = below + (above - below) / 2;
                    int mine[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < kMine; ++i)
                        mine[0] += a[i] > least ||
                                           (a[i] == least && ci[tid + i * kMergeThreads] <= upto)
                                       ? 1
                                       : 0;
                    total(mine, sum);
                    c = sum[0];
                    if (c < L)
                        below = upto;
                    else
                        above = upto;
                } while (!fits(c));
                break;
            }
            lo = nlo;
            hi = nhi;
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int e = tid + i * kMergeThreads;
            if (a[i] > least || (a[i] == least && ci[e] <= upto)) {
                const int pos = atomicAdd(&s_few, 1);
                few_s[pos] = a[i], few_i[pos] = ci[e];
            }
        }
        list_s = few_s;
        list_i = few_i;
        cnt = c;
        __syncthreads();
    }
    int nb;
    if (cnt <= CAND) {
        for (int c = tid; c < cnt; c += kMergeThreads) {
            const float s = list_s[c];
            const int i = list_i[c];
            int rank = 0;
            for (int j = 0; j < cnt; ++j) rank += ahead(list_s[j], list_i[j], s, i) ? 1 : 0;
            if (rank < L) bs[rank] = s, bi[rank] = i;
        }
        nb = min(L, cnt);
    } else {
        // more than CAND entries share the L-th best score: one arg-best a round
        float ls = INFINITY;
        int li = -1;
        for (nb = 0; nb < L; ++nb) {
            float b = -INFINITY;
            int bidx = INT_MAX;
            for (int e = tid; e < n_part * cap; e += kMergeThreads) {
                float s;
                int i;
                entry(e / cap, e % cap, s, i);
                if (i >= 0 && ahead(ls, li, s, i) && ahead(s, i, b, bidx)) b = s, bidx = i;
            }
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) {
                const float os = __shfl_xor_sync(0xffffffffu, b, o);
                const int oi = __shfl_xor_sync(0xffffffffu, bidx, o);
                if (ahead(os, oi, b, bidx)) b = os, bidx = oi;
            }
            __syncthreads();
            if (lane == 0) cs[warp] = b, ci[warp] = bidx;
            __syncthreads();
            for (int w = 0; w < kMergeThreads / 32; ++w)
                if (ahead(cs[w], ci[w], b, bidx)) b = cs[w], bidx = ci[w];
            if (bidx == INT_MAX) break;
            if (tid == 0) bs[nb] = b, bi[nb] = bidx;
            ls = b;
            li = bidx;
        }
    }
    __syncthreads();
    const double qq = s_qq;
    rescore(p, qv, qq, bi, nb, label, ex);
    __syncthreads();
    rank_candidates(ex, bi, nb, rank);
    __syncthreads();
    if (warp != 0) return;
    const int at = first_candidate(rank, nb);
    double M = 0.0, E = 0.0, S = 0.0;
    if (nb > 0) {
        M = ex[at];
        const double T = (double)p.temperature;
        float r0 = 0.0f, r1 = 0.0f;
        for (int w = 0; w < kMergeThreads / 32; ++w) r0 += red[0][w], r1 += red[1][w];
        r0 += (float)(s_ties - 1);
        const float d = (float)(T * ((double)ref - M)), f = expf(d);
        E = (double)(f * r0);
        S = (double)(f * (r1 * 0.69314718f + r0 * d));
        if (bs[at] != ref) {
            // the exact top is another score than the one left out
            const float b = (float)(T * ((double)bs[at] - M)), e = expf(b);
            E = fmax(E + (double)(f - e), 0.0);
            S += (double)(f * d - e * b);
        }
    }
    write_posterior(p, qi, bi, ex, nb, rank, !finite(qq), label, M, E, S);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Whether a pass over n_rows rows takes more than about half of the 126 MB L2.
int read_once(const RegDev& r, int n_rows) { return n_rows * r.row_bytes > (64LL << 20) ? 1 : 0; }

struct FewPlan {
    int nt, rows_per, n_slices, pitch, n_part;
    size_t smem;
};

// NT of a call: groups of 4 NT queries, each of which passes over the rows once. A group's
// rows are widened once for all its queries, but staging and selection go on query by query in
// every block, so small groups are better until a block has some 200 rows (of two an SM; 400
// for the step to 32 queries, 1000 where those leave room for one block an SM only), and 16
// queries stay where 32 would be padded by more than a quarter. Measured in us with 4, 8, 16
// and 32 queries a group, 8 bits:
//   posterior (k = 5), 256 dimensions   32 x 5000 rows 15 / 14 / 14 / 20, 32 x 20,000 31 / 17 /
//                      18 / 23, 64 x 20,000 31 / 23 / 21 / 26, 48 x 100,000 79 / 55 / 40 / 51
//   scores, 256 dimensions              32 x 1000 3.3 / 3.4 / 4.7 / 7.1, 64 x 5000 8.0 / 5.4 /
//                      6.1 / 7.2, 16 x 100,000 17 / 13 / 11 / 17, 32 x 100,000 30 / 21 / 18 / 18
int few_width(int n_rows, int n_q, int dim_pad) {
    int nt = 1;
    for (; nt < 8; nt *= 2) {
        const long long groups = (n_q + 4 * nt - 1) / (4 * nt), wide = (n_q + 8 * nt - 1) / (8 * nt);
        const long long most = nt < 4 ? 60000 : dim_pad <= 768 ? 120000 : 300000;
        if (groups == 1 || groups * n_rows <= most || (nt == 4 && 8 * wide > 5 * groups)) break;
    }
    return nt;
}

// Rows per block: two blocks an SM over all query groups, within what the block's score
// buffer (64 KB) and selection (a part a warp) take; at least 8 tiles.
FewPlan few_plan(const vdb_registry* r, int n_rows, int n_q, bool post) {
    FewPlan f{};
    // one query over 4-bit codes has a kernel of its own
    f.nt = n_q == 1 && r->bits == 4 ? 0 : few_width(n_rows, n_q, reg_dim_pad(r->dim));
    const int width = std::max(1, 4 * f.nt);
    const int nq = std::min(n_q, width);
    const long long groups = (n_q + width - 1) / width;
    // without a posterior nothing but 32-bit offsets into the block's rows limits them
    const int seg = post ? std::min(kFewMaxSeg, 16384 / nq / kPart * kPart) : 1 << 20;
    const long long blocks = 2LL * num_sms();
    const long long want = ((long long)n_rows * groups + blocks - 1) / blocks;
    f.rows_per = (int)std::max<long long>(128, std::min<long long>(seg, (want + 15) / 16 * 16));
    f.n_slices = (int)(((long long)n_rows + f.rows_per - 1) / f.rows_per);
    f.pitch = (f.rows_per + 31) / 32 * 32 + 8;
    f.smem = few_query_bytes(f.nt, reg_dim_pad(r->dim));
    if (post) {
        f.smem += (size_t)nq * f.pitch * 4;
        f.n_part = f.n_slices * ((f.rows_per + kPart - 1) / kPart);
    }
    return f;
}

template <int BITS, int NT, bool POST>
cudaError_t launch_few(const FewArgs& a, const FewPlan& f, cudaStream_t st) {
    auto kern = registry_few_kernel<BITS, NT, POST>;
    static SmemOptIn opt_in;  // of this instantiation
    if constexpr (POST && NT > 0) {
        // room for the larger merge's blocks beside these (k = 64, 12 queries x 100,000 rows: 57
        // us without, 41 with; the smaller one has it anyway, and the L1 is worth 2% there)
        const cudaError_t e = opt_in.carveout(kern, a.L > kMergeSmallL);
        if (e != cudaSuccess) return e;
    }
    if (f.smem > 48 * 1024) {
        const cudaError_t e = opt_in.allow(kern, f.smem);
        if (e != cudaSuccess) return e;
    }
    constexpr int width = NT ? 4 * NT : 1;
    const long long groups = (a.n_q + width - 1) / width;
    kern<<<(unsigned)(f.n_slices * groups), kFewThreads, f.smem, st>>>(a);
    return cudaGetLastError();
}

template <bool POST>
cudaError_t launch_few(int bits, const FewArgs& a, const FewPlan& f, cudaStream_t st) {
    if (bits == 8) {
        if (f.nt == 1) return launch_few<8, 1, POST>(a, f, st);
        if (f.nt == 2) return launch_few<8, 2, POST>(a, f, st);
        if (f.nt == 4) return launch_few<8, 4, POST>(a, f, st);
        return launch_few<8, 8, POST>(a, f, st);
    }
    if (f.nt == 0) return launch_few<4, 0, POST>(a, f, st);
    if (f.nt == 1) return launch_few<4, 1, POST>(a, f, st);
    if (f.nt == 2) return launch_few<4, 2, POST>(a, f, st);
    if (f.nt == 4) return launch_few<4, 4, POST>(a, f, st);
    return launch_few<4, 8, POST>(a, f, st);
}

// Whether the tensor cores' kernels, whose tiles hold 128 queries and which start with
// expanding the rows, take a call; otherwise the few-query kernel does. Measured at 256
// dimensions, 8 bits, few-query kernel / tensor cores, in us:
//   posterior (k = 5)  48 x 100,000 rows 40 / 57, 64 x 100,000 63 / 57, 128 x 20,000 31 / 31,
//                      300 x 5000 22 / 28, 600 x 5000 39 / 30
//   scores             64 x 100,000 28 / 30, 128 x 20,000 15 / 14, 128 x 100,000 49 / 38, 300 x
//                      5000 11 / 12, 600 x 5000 17 / 12
bool many_queries(int n_rows, int n_q, bool post) {
    return post ? (long long)(n_q - 32) * n_rows > 1900000
                : (long long)(n_q - 64) * n_rows > 1200000;
}

// The checks every entry point shares; false after setting the error.
bool check_registry(const char* who, const vdb_registry* r) {
    const auto fail = [&](const char* why) {
        set_error(std::string(who) + ": " + why);
        return false;
    };
    if (!r) return fail("NULL registry");
    if (r->capacity <= 0 || r->dim <= 0 || r->dim > kRegMaxDim)
        return fail("need capacity > 0, 0 < dim <= 1024");
    if (r->bits != 8 && r->bits != 4) return fail("bits must be 8 or 4");
    if (!r->codes || !r->scale || !r->owner || (r->bits == 4 && !r->group))
        return fail("NULL registry array");
    if (!aligned_to(r->codes, 16) || (r->bits == 4 && !aligned_to(r->group, 8)))
        return fail("codes need 16-byte, group 8-byte alignment");
    if (!aligned_to(r->scale, 4) || !aligned_to(r->owner, 4))
        return fail("scale and owner need 4-byte alignment");
    return true;
}

bool check_rows(const char* who, int type, const void* x, long long ld, int dim, int n) {
    const auto fail = [&](const char* why) {
        set_error(std::string(who) + ": " + why);
        return false;
    };
    if (type < kF32 || type > kBF16) return fail("element type must be 0 (f32), 1 (f16) or 2 (bf16)");
    if (n < 0) return fail("negative count");
    if (n > 0 && !x) return fail("NULL rows");
    if (n > 0 && !aligned_to(x, type == kF32 ? 4 : 2))
        return fail("rows need their element type's alignment");
    if (ld < dim) return fail("row pitch below dim");
    return true;
}

bool check_slots(const char* who, const vdb_registry* r, const int* slots, int first, int n) {
    if (n < 0) {
        set_error(std::string(who) + ": negative count");
        return false;
    }
    if (n > 0 && !aligned_to(slots, 4)) {
        set_error(std::string(who) + ": slots need 4-byte alignment");
        return false;
    }
    if (!slots && (first < 0 || (long long)first + n > r->capacity)) {
        set_error(std::string(who) + ": slots first .. first + n - 1 leave the registry");
        return false;
    }
    return true;
}

// The launch checks below are to see their own calls' errors only: one that another call of this
// library met and reported (an allocation that failed, say) is still the runtime's last one.
// Taken for a claim's, it would end a write half way and leave `owner` claimed.
void forget_errors() { (void)cudaGetLastError(); }

int finish(const char* who, cudaError_t e) {
    if (e == cudaSuccess) return 0;
    set_error(std::string(who) + ": " + cudaGetErrorString(e));
    return 1;
}

unsigned blocks_of(int n, int per) { return ((unsigned)n + (unsigned)per - 1) / (unsigned)per; }

template <typename T, int BITS>
cudaError_t launch_write(const vdb_registry* r, const void* x, long long ldx, const int* slots,
                         int first, int n, int* owner, cudaStream_t st) {
    const int dim_pad = reg_dim_pad(r->dim), nit = (dim_pad + 255) / 256;
    // rows that vector loads cannot take share the widest kernel
    const bool vec = aligned_to(x, 16) && ldx * sizeof(T) % 16 == 0 && r->dim % 8 == 0;
    auto kern = !vec       ? registry_write_kernel<T, BITS, 4, false>
                : nit == 1 ? registry_write_kernel<T, BITS, 1, true>
                : nit == 2 ? registry_write_kernel<T, BITS, 2, true>
                : nit == 3 ? registry_write_kernel<T, BITS, 3, true>
                           : registry_write_kernel<T, BITS, 4, true>;
    // few rows: one a warp, for the sake of latency
    const int per_warp = vec && n >= 64 * num_sms() ? write_rows(nit, sizeof(T) / 2) : 1;
    kern<<<blocks_of(n, 8 * per_warp), 256, 0, st>>>(
        static_cast<const T*>(x), ldx, slots, first, n, r->capacity, r->dim, dim_pad,
        reg_group_pitch(r->dim), (long long)dim_pad * BITS / 8, static_cast<uint8_t*>(r->codes),
        r->group, r->scale, owner, per_warp);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_write(const vdb_registry* r, const void* x, long long ldx, const int* slots,
                         int first, int n, int* owner, cudaStream_t st) {
    return r->bits == 8 ? launch_write<T, 8>(r, x, ldx, slots, first, n, owner, st)
                        : launch_write<T, 4>(r, x, ldx, slots, first, n, owner, st);
}

}  // namespace
}  // namespace vdb

using namespace vdb;

extern "C" int vdb_registry_dim_pad(int dim) {
    return dim > 0 && dim <= kRegMaxDim ? reg_dim_pad(dim) : 0;
}
extern "C" long long vdb_registry_row_bytes(int dim, int bits) {
    return (bits == 8 || bits == 4) ? (long long)vdb_registry_dim_pad(dim) * bits / 8 : 0;
}
extern "C" int vdb_registry_group_pitch(int dim) {
    return dim > 0 && dim <= kRegMaxDim ? reg_group_pitch(dim) : 0;
}

extern "C" int vdb_registry_clear(const vdb_registry* r, const int* slots, int first, int n,
                                  void* stream) {
    const char* who = "vdb_registry_clear";
    if (!check_registry(who, r) || !check_slots(who, r, slots, first, n)) return 1;
    if (n == 0) return 0;
    forget_errors();
    registry_clear_kernel<<<blocks_of(n, 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        r->scale, r->owner, r->capacity, slots, first, n);
    return finish(who, cudaGetLastError());
}

extern "C" int vdb_registry_write(const vdb_registry* r, const void* x, int x_type, long long ldx,
                                  const int* slots, int first, int n, void* stream) {
    const char* who = "vdb_registry_write";
    if (!check_registry(who, r) || !check_rows(who, x_type, x, ldx, r->dim, n) ||
        !check_slots(who, r, slots, first, n))
        return 1;
    if (n == 0) return 0;
    forget_errors();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int* owner = slots && n > 1 ? r->owner : nullptr;  // one row, or a range: no slot twice
    if (owner) {
        registry_claim_kernel<<<blocks_of(n, 256), 256, 0, st>>>(owner, r->capacity, slots, n);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return finish(who, e);
    }
    const cudaError_t e =
        x_type == kF32   ? launch_write<float>(r, x, ldx, slots, first, n, owner, st)
        : x_type == kF16 ? launch_write<__half>(r, x, ldx, slots, first, n, owner, st)
                         : launch_write<__nv_bfloat16>(r, x, ldx, slots, first, n, owner, st);
    return finish(who, e);
}

extern "C" int vdb_registry_read(const vdb_registry* r, const int* slots, int first, int n,
                                 void* out, int out_type, long long ldo, void* stream) {
    const char* who = "vdb_registry_read";
    if (!check_registry(who, r) || !check_rows(who, out_type, out, ldo, r->dim, n) ||
        !check_slots(who, r, slots, first, n))
        return 1;
    if (n == 0) return 0;
    forget_errors();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const RegDev d = reg_dev(r);
    const bool vec = aligned_to(out, 16) && ldo * (out_type == kF32 ? 4 : 2) % 16 == 0;
    const unsigned grid = blocks_of(n, 8);
    const auto go = [&](auto* o) {
        auto kern = r->bits == 8 ? registry_read_kernel<std::remove_pointer_t<decltype(o)>, 8>
                                 : registry_read_kernel<std::remove_pointer_t<decltype(o)>, 4>;
        kern<<<grid, 256, 0, st>>>(d, r->capacity, slots, first, n, o, ldo, vec);
    };
    if (out_type == kF32)
        go(static_cast<float*>(out));
    else if (out_type == kF16)
        go(static_cast<__half*>(out));
    else
        go(static_cast<__nv_bfloat16*>(out));
    return finish(who, cudaGetLastError());
}

extern "C" long long vdb_registry_score_work(const vdb_registry* r, int n_rows, int n_q) {
    if (!check_registry("vdb_registry_score_work", r)) return -1;
    if (n_rows < 0 || n_rows > r->capacity || n_q < 0) {
        set_error("vdb_registry_score_work: need 0 <= n_rows <= capacity, n_q >= 0");
        return -1;
    }
    return many_queries(n_rows, n_q, false) ? (long long)registry_tc_work(n_rows, n_q, r->dim, -1)
                                            : 0;
}

extern "C" int vdb_registry_score(const vdb_registry* r, int n_rows, const void* q, int q_type,
                                  long long ldq, int n_q, float* out, long long ldo, void* work,
                                  long long work_bytes, void* stream) {
    const char* who = "vdb_registry_score";
    if (!check_registry(who, r) || !check_rows(who, q_type, q, ldq, r->dim, n_q)) return 1;
    if (n_rows < 0 || n_rows > r->capacity || ldo < n_rows) {
        set_error("vdb_registry_score: need 0 <= n_rows <= capacity, ldo >= n_rows");
        return 1;
    }
    if (n_q == 0 || n_rows == 0) return 0;
    if (!out) {
        set_error("vdb_registry_score: NULL output");
        return 1;
    }
    if (!aligned_to(out, 4)) {
        set_error("vdb_registry_score: out needs 4-byte alignment");
        return 1;
    }
    forget_errors();
    const long long need = vdb_registry_score_work(r, n_rows, n_q);
    if (need > 0) {
        if (!work || work_bytes < need || !aligned_to(work, 256)) {
            set_error("vdb_registry_score: work: too small, NULL or not 256-byte aligned");
            return 1;
        }
        MergeArgs m{};
        m.r = reg_dev(r);
        m.n_rows = n_rows;
        m.q = q;
        m.q_type = q_type;
        m.ldq = ldq;
        m.n_q = n_q;
        return finish(who, registry_tc_run(m, -1, out, ldo, work, static_cast<cudaStream_t>(stream)));
    }
    const FewPlan f = few_plan(r, n_rows, n_q, false);
    FewArgs a{};
    a.r = reg_dev(r);
    a.r.once = read_once(a.r, n_rows);
    a.n_rows = n_rows;
    a.q = q;
    a.q_type = q_type;
    a.ldq = ldq;
    a.n_q = n_q;
    a.rows_per = f.rows_per;
    a.n_slices = f.n_slices;
    a.pitch = f.pitch;
    a.out = out;
    a.ldo = ldo;
    return finish(who, launch_few<false>(r->bits, a, f, static_cast<cudaStream_t>(stream)));
}

extern "C" long long vdb_registry_posterior_work(const vdb_registry* r, int n_rows, int n_q,
                                                 int k) {
    if (!check_registry("vdb_registry_posterior_work", r)) return -1;
    if (n_rows < 0 || n_rows > r->capacity || n_q < 0 || k < 0 || k > kRegMaxK) {
        set_error("vdb_registry_posterior_work: need 0 <= n_rows <= capacity, n_q >= 0, 0 <= k <= 64");
        return -1;
    }
    if (n_rows == 0 || n_q == 0) return 0;
    if (many_queries(n_rows, n_q, true)) return (long long)registry_tc_work(n_rows, n_q, r->dim, k);
    const FewPlan f = few_plan(r, n_rows, n_q, true);
    return (long long)reg_parts_bytes((size_t)f.n_part, (size_t)n_q, (size_t)list_size(k + kRegExtra));
}

extern "C" int vdb_registry_posterior(const vdb_registry* r, int n_rows, const void* q, int q_type,
                                      long long ldq, int n_q, float temperature, const int* labels,
                                      int k, float* log_prob, float* entropy, float* lse,
                                      int* alt_index, float* alt_log_prob, void* work,
                                      long long work_bytes, void* stream) {
    const char* who = "vdb_registry_posterior";
    if (!check_registry(who, r) || !check_rows(who, q_type, q, ldq, r->dim, n_q)) return 1;
    const auto fail = [&](const char* why) {
        set_error(std::string(who) + ": " + why);
        return 1;
    };
    if (n_rows < 0 || n_rows > r->capacity) return fail("need 0 <= n_rows <= capacity");
    if (k < 0 || k > kRegMaxK) return fail("need 0 <= k <= 64");
    if (!(temperature > 0.0f) || !(temperature <= 1e6f))
        return fail("temperature must be positive and at most 1e6");
    if ((labels != nullptr) != (log_prob != nullptr))
        return fail("labels and log_prob go together");
    if (n_q == 0) return 0;
    if (!entropy || !lse || (k > 0 && (!alt_index || !alt_log_prob))) return fail("NULL output");
    if (!aligned_to(labels, 4) || !aligned_to(log_prob, 4) || !aligned_to(entropy, 4) ||
        !aligned_to(lse, 4) || (k > 0 && (!aligned_to(alt_index, 4) || !aligned_to(alt_log_prob, 4))))
        return fail("labels and outputs need 4-byte alignment");
    const long long need = vdb_registry_posterior_work(r, n_rows, n_q, k);
    if (need > 0 && (!work || work_bytes < need || !aligned_to(work, 256)))
        return fail("work: too small, NULL or not 256-byte aligned");
    forget_errors();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int L = k + kRegExtra;
    MergeArgs m{};
    m.r = reg_dev(r);
    m.n_rows = n_rows;
    m.q = q;
    m.q_type = q_type;
    m.ldq = ldq;
    m.n_q = n_q;
    m.temperature = temperature;
    m.labels = labels;
    m.k = k;
    m.log_prob = log_prob;
    m.entropy = entropy;
    m.lse = lse;
    m.alt_index = alt_index;
    m.alt_log_prob = alt_log_prob;
    m.L = L;
    if (n_rows > 0 && many_queries(n_rows, n_q, true))
        return finish(who, registry_tc_run(m, k, nullptr, 0, work, st));
    if (n_rows > 0) {
        const FewPlan f = few_plan(r, n_rows, n_q, true);
        m.parts = reg_parts_at(work, (size_t)f.n_part, (size_t)n_q, (size_t)list_size(L));
        FewArgs a{};
        a.r = m.r;
        a.r.once = read_once(a.r, n_rows);
        a.n_rows = n_rows;
        a.q = q;
        a.q_type = q_type;
        a.ldq = ldq;
        a.n_q = n_q;
        a.rows_per = f.rows_per;
        a.n_slices = f.n_slices;
        a.pitch = f.pitch;
        a.s2 = temperature * 1.4426950408889634f;
        a.L = L;
        a.parts = m.parts;
        const cudaError_t e = launch_few<true>(r->bits, a, f, st);
        if (e != cudaSuccess) return finish(who, e);
    }
    auto merge = L <= kMergeSmallL ? registry_merge_kernel<1024> : registry_merge_kernel<2816>;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)n_q);
    cfg.blockDim = dim3(kMergeThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = n_rows > 0 ? 1 : 0;
    return finish(who, cudaLaunchKernelEx(&cfg, merge, m));
}
