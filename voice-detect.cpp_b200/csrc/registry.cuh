// Shared pieces of the quantised speaker registry's kernels (registry.cu,
// registry_tc.cu): the row layout, loads of the embedding types, the softmax partials and
// the candidate order. See vdb_ops.h for the stored format.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <climits>
#include <cstdint>
#include <cstring>
#include <mutex>

#include "sm100_ptx.cuh"
#include "vdb_internal.h"
#include "vdb_ops.h"

namespace vdb {

constexpr int kRegMaxDim = 1024;
constexpr int kRegMaxK = 64;
constexpr int kRegExtra = 4;  // candidates kept beyond k for the exact rescoring
// Unit query vectors are scaled by 2^8 before they are split into two f16: typical
// components (1/16 at 256 dims) become 16, so that the low part's rounding (up to 2^-23 of the
// component) stays clear of f16's subnormal step.
constexpr float kQScale = 256.0f;

__host__ __device__ inline int reg_dim_pad(int dim) { return (dim + 63) / 64 * 64; }
__host__ __device__ inline int reg_group_pitch(int dim) { return (dim + 255) / 256 * 8; }

enum : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

// Two packed f32: one instruction for both on sm_100.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack2(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(f2 v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// (score desc, slot asc): the order of candidates and of the alternatives.
__device__ __forceinline__ bool ahead(float s, int i, float t, int j) {
    return s > t || (s == t && i < j);
}

// The registry as the kernels see it.
struct RegDev {
    const uint8_t* codes;
    const uint8_t* group;
    const float* scale;
    int dim, dim_pad, gpitch, bits;
    long long row_bytes;
    int once;  // 1: a pass reads more than L2 keeps; its lines are the first to go
};

inline RegDev reg_dev(const vdb_registry* r) {
    RegDev d;
    d.codes = static_cast<const uint8_t*>(r->codes);
    d.group = r->group;
    d.scale = r->scale;
    d.dim = r->dim;
    d.dim_pad = reg_dim_pad(r->dim);
    d.gpitch = reg_group_pitch(r->dim);
    d.bits = r->bits;
    d.row_bytes = (long long)d.dim_pad * r->bits / 8;
    d.once = 0;
    return d;
}

// L2 eviction policy of a pass's code loads: a registry that L2 holds stays there between
// calls; a larger one must not push out everything else (the next kernel's code, the partials).
__device__ __forceinline__ uint64_t code_policy(int once) {
    uint64_t first, normal;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first));
    asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(normal));
    return once ? first : normal;
}
__device__ __forceinline__ uint4 load_codes16(const uint8_t* p, uint64_t policy) {
    uint4 v;
    asm("ld.global.nc.L1::no_allocate.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
        : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
        : "l"(p), "l"(policy));
    return v;
}
__device__ __forceinline__ uint2 load_codes8(const uint8_t* p, uint64_t policy) {
    uint2 v;
    asm("ld.global.nc.L1::no_allocate.L2::cache_hint.v2.u32 {%0, %1}, [%2], %3;"
        : "=r"(v.x), "=r"(v.y)
        : "l"(p), "l"(policy));
    return v;
}

// Softmax partials of one (part, query): the part's best score `ref` (a cosine; -inf: no
// score at all) and the sums over the part's other scores (one score equal to ref is left
// out) e0 = sum exp(temperature (c - ref)), e1 = the same times temperature (c - ref)
// log2 e. Leaving the best one out keeps a sum next to 0 from being lost under it.
// Candidate lists hold the part's best L scores and perhaps a few more (list_size), unordered,
// slot -1 past the last.
struct __align__(16) RegPart {
    float ref, e0, e1, pad;
};

struct RegParts {
    RegPart* stat;  // [n_part][n_q]
    float* score;   // [n_part][n_q][cap]
    int* slot;
    int n_part;
    int cap;  // entries a list
};

inline size_t reg_up(size_t b) { return (b + 255) / 256 * 256; }

inline size_t reg_parts_bytes(size_t n_part, size_t n_q, size_t cap) {
    return reg_up(n_part * n_q * sizeof(RegPart)) + 2 * reg_up(n_part * n_q * cap * 4);
}

inline RegParts reg_parts_at(void* work, size_t n_part, size_t n_q, size_t cap) {
    RegParts p;
    uint8_t* w = static_cast<uint8_t*>(work);
    p.stat = reinterpret_cast<RegPart*>(w);
    w += reg_up(n_part * n_q * sizeof(RegPart));
    p.score = reinterpret_cast<float*>(w);
    w += reg_up(n_part * n_q * cap * 4);
    p.slot = reinterpret_cast<int*>(w);
    p.n_part = (int)n_part;
    p.cap = (int)cap;
    return p;
}

constexpr int kPart = 512;  // scores one warp selects from: 16 a lane

// The whole numbers of 8 consecutive dimensions (d0 a multiple of 8) of one row.
__device__ __forceinline__ void whole8(const uint8_t* codes, const uint8_t* group, int bits,
                                       int d0, int (&w)[8]) {
    if (bits == 8) {
        const uint2 c = *reinterpret_cast<const uint2*>(codes + d0);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            w[j] = (int)(((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 255u) - 128;
    } else {
        const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + d0 / 2);
        const int s = group[d0 >> 5];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            w[j] = ((int)((c >> (4 * ((j >> 1) + (j & 1) * 4))) & 15u) - 8) * s;
    }
}

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
    __half2 x, y;
    memcpy(&x, &a, 4);
    memcpy(&y, &b, 4);
    x = __hsub2(x, y);
    uint32_t r;
    memcpy(&r, &x, 4);
    return r;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
    __half2 x, y, z;
    memcpy(&x, &a, 4);
    memcpy(&y, &b, 4);
    memcpy(&z, &c, 4);
    x = __hfma2(x, y, z);
    uint32_t r;
    memcpy(&r, &x, 4);
    return r;
}

// Four byte codes w + 128 -> the whole numbers w as two f16 pairs: the byte in the low
// mantissa bits of 1024.0 is 1024 + w + 128, and the subtraction is exact.
__device__ __forceinline__ void widen8(uint32_t x, uint32_t& p0, uint32_t& p1) {
    p0 = h2_sub(__byte_perm(x, 0x64646464u, 0x4140), 0x64806480u);
    p1 = h2_sub(__byte_perm(x, 0x64646464u, 0x4342), 0x64806480u);
}

// Eight nibble codes c + 8 of one group -> c s as four f16 pairs in dimension order: a
// nibble in mantissa bits 4-7 of 64.0 is 64 + c + 8; times s, minus 72 s, in one fused
// step whose result (at most 889) is exact. 72 s = 8 (9 s) <= 9144 is exact too.
__device__ __forceinline__ void widen4(uint32_t x, uint32_t s, uint32_t ms, uint32_t (&p)[4]) {
    p[0] = h2_fma(((x << 4) & 0x00F000F0u) | 0x54005400u, s, ms);
    p[1] = h2_fma((x & 0x00F000F0u) | 0x54005400u, s, ms);
    p[2] = h2_fma(((x >> 4) & 0x00F000F0u) | 0x54005400u, s, ms);
    p[3] = h2_fma(((x >> 8) & 0x00F000F0u) | 0x54005400u, s, ms);
}

// 256 dimensions (four chunks of 64 from c0 on) of two rows as one lane of an m16n8k16
// operand holds them: 16 consecutive dimensions 16 t .. 16 t + 15 of each chunk.
template <int BITS>
struct RowFrag {
    uint4 xa[4], xb[4];
    uint2 sa, sb;  // 4 bits: the eight group scales of the 256 dimensions

    __device__ __forceinline__ void load(const RegDev& r, long long ra, long long rb, int c0,
                                         int n_chunks, int t, uint64_t policy) {
        const uint8_t* ca = r.codes + ra * r.row_bytes;
        const uint8_t* cb = r.codes + rb * r.row_bytes;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            xa[u] = xb[u] = make_uint4(0u, 0u, 0u, 0u);
            if (c0 + u >= n_chunks) continue;
            if constexpr (BITS == 8) {
                xa[u] = load_codes16(ca + (c0 + u) * 64 + 16 * t, policy);
                xb[u] = load_codes16(cb + (c0 + u) * 64 + 16 * t, policy);
            } else {
                const uint2 va = load_codes8(ca + (c0 + u) * 32 + 8 * t, policy);
                const uint2 vb = load_codes8(cb + (c0 + u) * 32 + 8 * t, policy);
                xa[u].x = va.x, xa[u].y = va.y;
                xb[u].x = vb.x, xb[u].y = vb.y;
            }
        }
        if constexpr (BITS == 4) {
            sa = __ldg(reinterpret_cast<const uint2*>(r.group + ra * r.gpitch) + c0 / 4);
            sb = __ldg(reinterpret_cast<const uint2*>(r.group + rb * r.gpitch) + c0 / 4);
        }
    }

    // Chunk c0 + u as f16 pairs of dimensions 2i, 2i + 1 of the lane's 16.
    __device__ __forceinline__ void widen(int u, int t, uint32_t (&fa)[8],
                                          uint32_t (&fb)[8]) const {
        if constexpr (BITS == 8) {
            widen8(xa[u].x, fa[0], fa[1]);
            widen8(xa[u].y, fa[2], fa[3]);
            widen8(xa[u].z, fa[4], fa[5]);
            widen8(xa[u].w, fa[6], fa[7]);
            widen8(xb[u].x, fb[0], fb[1]);
            widen8(xb[u].y, fb[2], fb[3]);
            widen8(xb[u].z, fb[4], fb[5]);
            widen8(xb[u].w, fb[6], fb[7]);
        } else {
            // the lane's group scale: byte 2u + t / 2 of the 256 dimensions' eight
            const uint32_t sel = 0x4040u + 0x0101u * (uint32_t)((u & 1) * 2 + (t >> 1));
            const uint32_t m1024 = 0x64006400u, m72 = 0xD480D480u;  // 1024, -72
            const uint32_t s_a = h2_sub(__byte_perm(u < 2 ? sa.x : sa.y, 0x64646464u, sel), m1024);
            const uint32_t s_b = h2_sub(__byte_perm(u < 2 ? sb.x : sb.y, 0x64646464u, sel), m1024);
            const uint32_t ms_a = h2_fma(s_a, m72, 0u), ms_b = h2_fma(s_b, m72, 0u);
            uint32_t w[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                widen4(h ? xa[u].y : xa[u].x, s_a, ms_a, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) fa[4 * h + i] = w[i];
                widen4(h ? xb[u].y : xb[u].x, s_b, ms_b, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) fb[4 * h + i] = w[i];
            }
        }
    }
};

// Eight consecutive values of an embedding row as f32, 0 past `left`; one vector load each
// where the row allows it.
__device__ __forceinline__ void emb8(const void* base, int type, long long i, int left,
                                     float (&v)[8]) {
    if (type == kF32) {
        const float* p = static_cast<const float*>(base) + i;
        if (left >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
            const float4 a = *reinterpret_cast<const float4*>(p);
            const float4 b = *reinterpret_cast<const float4*>(p + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
            v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.0f;
        return;
    }
    const uint16_t* p = static_cast<const uint16_t*>(base) + i;
    uint32_t w[4];
    if (left >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = (2 * j < left ? (uint32_t)p[2 * j] : 0u) |
                   (2 * j + 1 < left ? (uint32_t)p[2 * j + 1] << 16 : 0u);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (type == kF16) {
            v[2 * j] = __half2float(__ushort_as_half((unsigned short)(w[j] & 0xFFFFu)));
            v[2 * j + 1] = __half2float(__ushort_as_half((unsigned short)(w[j] >> 16)));
        } else {  // bf16 is the upper half of an f32
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
    }
}

// One query's row by one warp: up to 512 dimensions in registers (the rest is loaded again
// where it is needed), its squared length in f64 (no overflow, no loss for very long or short
// queries) and its largest |component| (an infinity or a NaN: 0x7F800000 or more).
struct QueryRow {
    static constexpr int kKeep = 2;
    float v[kKeep][8];
    double square;
    uint32_t most;

    __device__ __forceinline__ void load(const void* q, int q_type, long long row0, int dim) {
        const int lane = threadIdx.x & 31;
        double s0 = 0.0, s1 = 0.0;
        most = 0;
        const auto add = [&](const float(&x)[8]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s0 += (double)x[j] * (double)x[j];
                s1 += (double)x[j + 4] * (double)x[j + 4];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(x[j]) & 0x7FFFFFFFu);
        };
#pragma unroll
        for (int it = 0; it < kKeep; ++it) {
            const int d0 = it * 256 + lane * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[it][j] = 0.0f;
            if (d0 < dim) emb8(q, q_type, row0 + d0, dim - d0, v[it]);
        }
#pragma unroll
        for (int it = 0; it < kKeep; ++it) add(v[it]);
        for (int d0 = kKeep * 256 + lane * 8; d0 < dim; d0 += 256) {
            float x[8];
            emb8(q, q_type, row0 + d0, dim - d0, x);
            add(x);
        }
        s0 += s1;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
        square = s0;
        most = __reduce_max_sync(0xffffffffu, most);
    }
    // put(d0, x) for the lane's eights of d0 < dim_pad (zeros past dim)
    template <typename Put>
    __device__ __forceinline__ void each(const void* q, int q_type, long long row0, int dim,
                                         int dim_pad, Put put) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int it = 0; it < kKeep; ++it) {
            const int d0 = it * 256 + lane * 8;
            if (d0 < dim_pad) put(d0, v[it]);
        }
        for (int d0 = kKeep * 256 + lane * 8; d0 < dim_pad; d0 += 256) {
            float x[8] = {};
            if (d0 < dim) emb8(q, q_type, row0 + d0, dim - d0, x);
            put(d0, x);
        }
    }
};

// A power of two that brings numbers of size x (or 1 / x) near enough to 1 for f32 factors.
__device__ __forceinline__ float near_one(double x) {
    return x > 0x1p100 ? 0x1p-100f : x < 0x1p-100 ? 0x1p100f : 1.0f;
}

// One query's unit vector as f16 high and low parts (of kQScale times it), by one warp;
// zeros for a zero query and past dim, handed to put(d0, hi, lo) as eight f16 each from
// dimension d0. The parts are off by up to 2^-23 of a component (the high one by 2^-12 of its
// power of two, the low one by as much of its own), which is what the vector's f32 roundings
// cost. A query with an infinity or a NaN gives NaNs (rsqrt(inf) = 0, and 0 * inf = NaN).
template <typename Put>
__device__ __forceinline__ void split_query(const void* q, int q_type, long long row0, int dim,
                                            int dim_pad, bool present, Put put) {
    QueryRow r;
    r.load(q, q_type, row0, present ? dim : 0);
    const double n = rsqrt(r.square);
    const float near = r.square == 0.0 ? 1.0f : near_one(n);  // a power of two
    const float pre = near < 1.0f ? 0x1p100f : near > 1.0f ? 0x1p-100f : 1.0f;  // 1 / near
    const float inv = r.square == 0.0 ? 0.0f : (float)((double)kQScale * n * (double)near);
    r.each(q, q_type, row0, present ? dim : 0, dim_pad, [&](int d0, const float(&x)[8]) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = x[2 * j] * pre * inv, b = x[2 * j + 1] * pre * inv;
            const __half2 ab = __floats2half2_rn(a, b);
            const float2 f = __half22float2(ab);
            const __half2 cd = __floats2half2_rn(a - f.x, b - f.y);
            memcpy(&h[j], &ab, 4);
            memcpy(&l[j], &cd, 4);
        }
        put(d0, h, l);
    });
}

// One query in fixed point, by one warp: component x as x 2^23 / max|x| = 2^12 hi + lo with
// whole numbers |hi|, |lo| <= 2048, f16 each (exact): 2^-24 of the largest component where two
// rounded f16 parts keep 2^-23 of each, so that what is lost is an f32 product's error.
// Returns what 2^12 hi + lo is to be multiplied with to give the unit vector, on every lane
// (NaN for a query with an infinity or a NaN).
template <typename Put>
__device__ __forceinline__ float split_query_fixed(const void* q, int q_type, long long row0,
                                                   int dim, int dim_pad, Put put) {
    QueryRow r;
    r.load(q, q_type, row0, dim);
    const bool bad = r.most >= 0x7F800000u;
    const float top = __uint_as_float(bad ? 0u : r.most);
    const float pre = top > 0.0f ? near_one((double)top) : 1.0f;
    const float f = top > 0.0f ? 8388608.0f / (top * pre) : 0.0f;
    r.each(q, q_type, row0, dim, dim_pad, [&](int d0, const float(&x)[8]) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = bad ? 0.0f : x[2 * j] * pre * f;
            const float b = bad ? 0.0f : x[2 * j + 1] * pre * f;
            const float ha = rintf(a * (1.0f / 4096.0f)), hb = rintf(b * (1.0f / 4096.0f));
            const __half2 ab = __floats2half2_rn(ha, hb);
            const __half2 cd = __floats2half2_rn(rintf(fmaf(ha, -4096.0f, a)),
                                                 rintf(fmaf(hb, -4096.0f, b)));
            memcpy(&h[j], &ab, 4);
            memcpy(&l[j], &cd, 4);
        }
        put(d0, h, l);
    });
    if (bad) return __int_as_float(0x7FC00000);
    return top > 0.0f ? (float)((double)top * rsqrt(r.square) * 0x1p-23) : 0.0f;
}

// The parts into two rows of memory.
struct StoreParts {
    __half *hi, *lo;
    __device__ __forceinline__ void operator()(int d0, const uint32_t (&h)[4],
                                               const uint32_t (&l)[4]) const {
        *reinterpret_cast<uint4*>(hi + d0) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(lo + d0) = make_uint4(l[0], l[1], l[2], l[3]);
    }
};

__device__ __forceinline__ float h2_sum(uint32_t v) {
    __half2 h;
    memcpy(&h, &v, 4);
    const float2 f = __half22float2(h);
    return f.x + f.y;
}

// Order-preserving map of a float to an unsigned key (-0 maps to 0's key).
__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t b = __float_as_uint(f + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float from_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// The L-th largest (L <= 32) of the lanes' keys, 0 when fewer than L are above 0: the lanes'
// keys sorted by a bitonic network, whose 15 exchanges take a third of the time of L rounds of
// a warp maximum.
__device__ __forceinline__ uint32_t lth_lane_key(uint32_t key, int L) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int run = 2; run <= 32; run <<= 1)
#pragma unroll
        for (int o = run / 2; o >= 1; o >>= 1) {
            const uint32_t x = __shfl_xor_sync(0xffffffffu, key, o);
            // descending runs where bit `run` of the lane is clear
            key = ((lane & run) == 0) == ((lane & o) == 0) ? max(key, x) : min(key, x);
        }
    return __shfl_sync(0xffffffffu, key, L - 1);
}

// The L-th largest (L <= 32 N) of N keys a lane, by one warp: the largest key that at least L
// of them reach, 0 when there are fewer than L keys above 0.
template <int N>
__device__ __forceinline__ uint32_t lth_key(const uint32_t (&key)[N], int L) {
    uint32_t bound = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
        const uint32_t tr = bound | (1u << b);
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += __popc(__ballot_sync(0xffffffffu, key[i] >= tr));
        if (n >= L) bound = tr;
    }
    return bound;
}

// Entries of a candidate list: L, or a few more where that saves looking for exactly L.
__host__ __device__ constexpr int list_size(int L) { return (L + 9) / 2 * 2; }

// The best L of n <= 32 S scores (shared memory; slots `slot[i]`, or base + i), by one warp,
// or up to cap >= L that hold them, written to out_s / out_i in any order (slot -1 past the
// last of cap), and the part's sums. A bound that L to cap scores reach: for L <= 12 the L-th
// largest of the 32 lane maxima (at least L reach it, mostly few more), otherwise by
// bisection between the least and the largest score. Where ties leave no such bound, L
// rounds of an arg-best over the warp.
template <int S>
__device__ __forceinline__ RegPart warp_select(const float* v, const int* slot, int base, int n,
                                               int L, int cap, float s2, float* out_s, int* out_i) {
    const int lane = threadIdx.x & 31;
    constexpr unsigned full = 0xffffffffu;
    float a[S];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int e = lane + 32 * i;
        a[i] = e < n ? v[e] : -INFINITY;
        m = fmaxf(m, a[i]);
    }
    RegPart out{m, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) out.ref = fmaxf(out.ref, __shfl_xor_sync(full, out.ref, o));
    uint32_t mine = 0;  // this lane's scores that reach the bound
    int cnt = 0, filled = 0;
    const auto reach = [&](float bound) {
        mine = 0;
#pragma unroll
        for (int i = 0; i < S; ++i) mine |= a[i] >= bound ? 1u << i : 0u;
        cnt = __reduce_add_sync(full, __popc(mine));
        return cnt;
    };
    bool done = out.ref == -INFINITY;
    if (!done) {
        if (L <= 12) {
            const uint32_t low = lth_lane_key(m > -INFINITY ? key_of(m) : 0u, L);
            done = reach(low == 0 ? -FLT_MAX : from_key(low)) <= cap;
        }
        if (!done) done = reach(-FLT_MAX) <= cap;
        if (!done) {
            float lo = INFINITY, hi = out.ref;
#pragma unroll
            for (int i = 0; i < S; ++i) lo = a[i] > -INFINITY ? fminf(lo, a[i]) : lo;
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) lo = fminf(lo, __shfl_xor_sync(full, lo, o));
            // more than cap reach lo
            while (!done) {
                const float mid = 0.5f * lo + 0.5f * hi;
                const bool last = !(mid > lo && mid < hi);
                const int c = reach(last ? hi : mid);
                done = c >= L && c <= cap;
                if (last) break;
                if (c > cap)
                    lo = mid;
                else
                    hi = mid;
            }
        }
    }
    if (done) {
        int pos = __popc(mine);
        const int own = pos;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(full, pos, o);
            pos += lane >= o ? x : 0;
        }
        pos -= own;
        for (; mine; mine &= mine - 1, ++pos) {
            const int e = lane + 32 * (__ffs(mine) - 1);
            out_s[pos] = v[e];
            out_i[pos] = slot ? slot[e] : base + e;
        }
        filled = cnt;
    } else {
        uint32_t taken = 0;
        for (filled = 0; filled < L; ++filled) {
            float bs = -INFINITY;
            int bi = INT_MAX, bp = 0;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const int e = lane + 32 * i;
                if (((taken >> i) & 1) || !(a[i] > -INFINITY)) continue;
                const int si = slot ? slot[e] : base + e;
                if (ahead(a[i], si, bs, bi)) {
                    bs = a[i];
                    bi = si;
                    bp = i;
                }
            }
            float ws = bs;
            int wi = bi;
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) {
                const float os = __shfl_xor_sync(full, ws, o);
                const int oi = __shfl_xor_sync(full, wi, o);
                if (ahead(os, oi, ws, wi)) {
                    ws = os;
                    wi = oi;
                }
            }
            if (wi == INT_MAX) break;
            if (bi == wi) {
                taken |= 1u << bp;
                out_s[filled] = ws;
                out_i[filled] = wi;
            }
        }
    }
    for (int j = filled + lane; j < cap; j += 32) {
        out_s[j] = -INFINITY;
        out_i[j] = -1;
    }
    __syncwarp();
    if (out.ref == -INFINITY) return out;
    int ties = 0;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        if (32 * i >= n) break;
        // NaN scores are a non-finite query's: its sums are not looked at
        const bool at_top = a[i] == out.ref;
        const float t = (a[i] - out.ref) * s2, ex = exp2f(t);  // 0 for an empty slot
        ties += at_top ? 1 : 0;
        out.e0 += at_top ? 0.0f : ex;
        out.e1 += a[i] > -INFINITY ? ex * t : 0.0f;
    }
    ties = __reduce_add_sync(full, ties);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        out.e0 += __shfl_xor_sync(full, out.e0, o);
        out.e1 += __shfl_xor_sync(full, out.e1, o);
    }
    out.e0 += (float)(ties - 1);
    return out;
}

// What the kernels that end in a posterior read and write.
struct MergeArgs {
    RegDev r;
    int n_rows;
    const void* q;
    int q_type;
    long long ldq;
    int n_q;
    float temperature;
    const int* labels;
    int k;
    float *log_prob, *entropy, *lse;
    int* alt_index;
    float* alt_log_prob;
    RegParts parts;
    int L;  // candidates wanted: k + kRegExtra
};

// The query in f64 in shared memory (dim_pad values, zeros past dim) and its |q|^2, by one
// warp (every lane gets the sum). Dimension 64 i + 8 l + j is entry 64 i + 16 (j / 2) + 2 l +
// j % 2, so that eight lanes l read a pair each from neighbouring 16 bytes.
__device__ __forceinline__ double stage_query(const MergeArgs& p, int qi, double* qv) {
    const int lane = threadIdx.x & 31;
    double s = 0.0;
    for (int d0 = lane * 8; d0 < p.r.dim_pad; d0 += 256) {
        float v[8];
        emb8(p.q, p.q_type, (long long)qi * p.ldq + d0, p.r.dim - d0, v);
        double2* o = reinterpret_cast<double2*>(qv + (d0 & ~63)) + ((d0 >> 3) & 7);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[8 * j] = make_double2((double)v[2 * j], (double)v[2 * j + 1]);
            s += (double)v[2 * j] * (double)v[2 * j] + (double)v[2 * j + 1] * (double)v[2 * j + 1];
        }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

__device__ __forceinline__ bool finite(double v) { return v <= 1.7976931348623157e308; }

// The query's label's slot, -1 when there is none or it is not enrolled.
__device__ __forceinline__ int label_of(const MergeArgs& p, int qi) {
    int label = p.labels ? p.labels[qi] : -1;
    if (label >= p.n_rows || (label >= 0 && !(p.r.scale[label] == p.r.scale[label]))) label = -1;
    return label;
}

// Eight consecutive dimensions (d0 a multiple of 8) of one row times those of a query: adds to
// the dot product and to the sum of squares. The query's pairs are at v[0], v[8], v[16], v[24].
__device__ __forceinline__ void exact8(const uint8_t* codes, const uint8_t* group, int bits, int d0,
                                       const double2* v, double& dot, int& w2) {
    if (bits == 8) {
        uint2 c = *reinterpret_cast<const uint2*>(codes + d0);
        c.x ^= 0x80808080u;  // w as signed bytes
        c.y ^= 0x80808080u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t x = (j < 2 ? c.x : c.y) >> (16 * (j & 1));
            const double2 q = v[8 * j];
            dot += q.x * (double)(int8_t)(x & 255u);
            dot += q.y * (double)(int8_t)((x >> 8) & 255u);
        }
        w2 = __dp4a((int)c.x, (int)c.x, w2);
        w2 = __dp4a((int)c.y, (int)c.y, w2);
    } else {
        const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + d0 / 2) ^ 0x88888888u;
        const int s = group[d0 >> 5];
        double part = 0.0;
        int sq = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // dimensions 2j and 2j + 1: nibbles j and j + 4, signed
            const int a = (int)(c << (28 - 4 * j)) >> 28, b = (int)(c << (12 - 4 * j)) >> 28;
            const double2 q = v[8 * j];
            part += q.x * (double)a;
            part += q.y * (double)b;
            sq += a * a + b * b;
        }
        dot += part * (double)s;
        w2 += sq * s * s;
    }
}

// Exact (f64) cosines of the nb candidates `slots` and, as entry nb, of the label's slot, by
// all warps of the block, eight lanes a candidate. qv, qq: stage_query's. The caller
// synchronises.
__device__ __forceinline__ void rescore(const MergeArgs& p, const double* qv, double qq,
                                        const int* slots, int nb, int label, double* ex) {
    const int lane = threadIdx.x & 31, l = lane & 7;
    const int n = nb + (label >= 0 ? 1 : 0);
    for (int c0 = (threadIdx.x >> 5) * 4; c0 < n; c0 += blockDim.x / 8) {
        const int c = c0 + (lane >> 3);
        const long long slot = c < nb ? slots[c] : c < n ? label : 0;
        const uint8_t* codes = p.r.codes + slot * p.r.row_bytes;
        const uint8_t* group = p.r.group + slot * p.r.gpitch;
        double dot = 0.0;
        int w2 = 0;
#pragma unroll 4
        for (int i = 0; i < p.r.dim_pad; i += 64)
            exact8(codes, group, p.r.bits, i + 8 * l,
                   reinterpret_cast<const double2*>(qv + i) + l, dot, w2);
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) {
            dot += __shfl_xor_sync(0xffffffffu, dot, o);
            w2 += __shfl_xor_sync(0xffffffffu, w2, o);
        }
        const double den = sqrt(qq * (double)w2);
        if (l == 0 && c < n) ex[c] = den > 0.0 ? dot / den : 0.0;
    }
}

// The candidates' order by (cosine rounded to f32, lower slot), by all threads of the block:
// rank[c] of candidate c. The caller synchronises.
__device__ __forceinline__ void rank_candidates(const double* ex, const int* slots, int nb,
                                                int* rank) {
    for (int c = threadIdx.x; c < nb; c += blockDim.x) {
        const float f = (float)ex[c];
        const int s = slots[c];
        int n = 0;
#pragma unroll 4
        for (int j = 0; j < nb; ++j) n += ahead((float)ex[j], slots[j], f, s) ? 1 : 0;
        rank[c] = n;
    }
}

// The candidate of rank 0, by one warp.
__device__ __forceinline__ int first_candidate(const int* rank, int nb) {
    int first = INT_MAX;
    for (int c = threadIdx.x & 31; c < nb; c += 32)
        if (rank[c] == 0) first = c;
    return (int)__reduce_min_sync(0xffffffffu, (unsigned)first);
}

// Writes a query's results, by one warp: M is the top candidate's cosine, E and S are the sums
// of e = exp(temperature (c - M)) and of e temperature (c - M) over every score c but that
// one; rank: rank_candidates'.
__device__ __forceinline__ void write_posterior(const MergeArgs& p, int qi, const int* slots,
                                                const double* ex, int nb, const int* rank,
                                                bool bad, int label, double M, double E, double S) {
    const int lane = threadIdx.x & 31;
    const bool none = nb == 0;
    // (f32: its result is rounded to f32 anyway, and its relative error is that of an f32)
    const double T = (double)p.temperature, lg = (double)log1pf((float)E);
    const float nan = __int_as_float(0x7FC00000);
    if (lane == 0) {
        p.lse[qi] = bad ? nan : none ? -INFINITY : (float)(T * M + lg);
        p.entropy[qi] = bad ? nan : none ? 0.0f : (float)lg - (float)S / (1.0f + (float)E);
        if (p.log_prob) {
            float v = -INFINITY;
            if (label >= 0 && !none) v = (float)fmin(0.0, T * (ex[nb] - M) - lg);
            p.log_prob[qi] = bad ? nan : v;
        }
    }
    for (int j = lane; j < p.k; j += 32) {
        if (j >= nb || bad) {
            p.alt_index[(long long)qi * p.k + j] = -1;
            p.alt_log_prob[(long long)qi * p.k + j] = -INFINITY;
        }
    }
    if (bad) return;
    for (int c = lane; c < nb; c += 32) {
        if (rank[c] >= p.k) continue;
        p.alt_index[(long long)qi * p.k + rank[c]] = slots[c];
        p.alt_log_prob[(long long)qi * p.k + rank[c]] = (float)(T * (ex[c] - M) - lg);
    }
}

// What each device has been asked for one kernel: the largest dynamic shared memory to allow,
// and whether all that can be shared memory is to be.
struct SmemOptIn {
    std::mutex mu;
    size_t set[64] = {};
    bool wide[64] = {};
    template <typename K>
    cudaError_t carveout(K kern, bool most) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (dev < 0 || dev >= 64) return cudaSuccess;  // (it only costs time)
        std::lock_guard<std::mutex> lk(mu);
        if (wide[dev] == most) return cudaSuccess;
        wide[dev] = most;
        return cudaFuncSetAttribute(
            kern, cudaFuncAttributePreferredSharedMemoryCarveout,
            most ? cudaSharedmemCarveoutMaxShared : cudaSharedmemCarveoutDefault);
    }
    template <typename K>
    cudaError_t allow(K kern, size_t bytes) {
        int dev = 0;
        cudaGetDevice(&dev);
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 0 && dev < 64 && set[dev] >= bytes) return cudaSuccess;
        const cudaError_t e = cudaFuncSetAttribute(
            kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess && dev >= 0 && dev < 64) set[dev] = bytes;
        return e;
    }
};

// ---- the tensor-core path for many queries (registry_tc.cu) ----
// Bytes of working memory, and the launches: scores into out (k < 0) or a posterior.
size_t registry_tc_work(int n_rows, int n_q, int dim, int k);
cudaError_t registry_tc_run(const MergeArgs& m, int k, float* out, long long ldo, void* work,
                            cudaStream_t st);

}  // namespace vdb
