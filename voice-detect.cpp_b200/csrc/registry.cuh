// Shared pieces of the quantised speaker registry's kernels (registry.cu,
// registry_tc.cu): the row layout, loads of the embedding types, the softmax partials and
// the candidate order. See vdb_ops.h for the stored format.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
constexpr int kRegExtra = 8;  // candidates kept beyond k for the exact rescoring
// Unit query vectors are scaled by 2^8 before they are split into two f16: typical
// components (1/16 at 256 dims) become 16, so that the low part's rounding (2^-25 of the
// component) stays clear of f16's subnormal step.
constexpr float kQScale = 256.0f;

__host__ __device__ inline int reg_dim_pad(int dim) { return (dim + 63) / 64 * 64; }
__host__ __device__ inline int reg_group_pitch(int dim) { return (dim + 255) / 256 * 8; }

enum : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float load_emb(const void* base, int type, long long i) {
    if (type == kF32) return static_cast<const float*>(base)[i];
    if (type == kF16) return __half2float(static_cast<const __half*>(base)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
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
    return d;
}

// Softmax partials of one (part, query): the sums over the part's scores that are not in
// its candidate list, relative to the list's best score `ref` (-inf: no score at all):
// e0 = sum exp(temperature (c - ref)), e1 = the same times temperature (c - ref) log2 e.
// Lists hold L entries, unordered, slot -1 past the last.
struct RegPart {
    float ref, e0, e1;
};

struct RegParts {
    RegPart* stat;  // [n_part][n_q]
    float* score;   // [n_part][n_q][L]
    int* slot;
    int n_part;
    int L;
};

inline size_t reg_up(size_t b) { return (b + 255) / 256 * 256; }

inline size_t reg_parts_bytes(size_t n_part, size_t n_q, size_t L) {
    return reg_up(n_part * n_q * sizeof(RegPart)) + 2 * reg_up(n_part * n_q * L * 4);
}

inline RegParts reg_parts_at(void* work, size_t n_part, size_t n_q, size_t L) {
    RegParts p;
    uint8_t* w = static_cast<uint8_t*>(work);
    p.stat = reinterpret_cast<RegPart*>(w);
    w += reg_up(n_part * n_q * sizeof(RegPart));
    p.score = reinterpret_cast<float*>(w);
    w += reg_up(n_part * n_q * L * 4);
    p.slot = reinterpret_cast<int*>(w);
    p.n_part = (int)n_part;
    p.L = (int)L;
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
                                         int n_chunks, int t) {
        const uint8_t* ca = r.codes + ra * r.row_bytes;
        const uint8_t* cb = r.codes + rb * r.row_bytes;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            xa[u] = xb[u] = make_uint4(0u, 0u, 0u, 0u);
            if (c0 + u >= n_chunks) continue;
            if constexpr (BITS == 8) {
                xa[u] = __ldg(reinterpret_cast<const uint4*>(ca + (c0 + u) * 64) + t);
                xb[u] = __ldg(reinterpret_cast<const uint4*>(cb + (c0 + u) * 64) + t);
            } else {
                const uint2 va = __ldg(reinterpret_cast<const uint2*>(ca + (c0 + u) * 32) + t);
                const uint2 vb = __ldg(reinterpret_cast<const uint2*>(cb + (c0 + u) * 32) + t);
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

// One query's unit vector as f16 high and low parts (of kQScale times it) into two rows of
// shared memory, by one warp; zeros for a zero query and past dim.
__device__ __forceinline__ void split_query(const void* q, int q_type, long long row0, int dim, int dim_pad,
                            bool present, __half* hi, __half* lo) {
    const int lane = threadIdx.x & 31;
    double s = 0.0;
    if (present)
        for (int d = lane; d < dim; d += 32) {
            const double v = load_emb(q, q_type, row0 + d);
            s += v * v;
        }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    // a NaN or infinite norm stays one: inf * 0 and NaN make the whole vector NaN
    const double inv = s == 0.0 ? 0.0 : (double)kQScale / sqrt(s);
    for (int d = lane; d < dim_pad; d += 32) {
        const double v = present && d < dim ? (double)load_emb(q, q_type, row0 + d) * inv : 0.0;
        const __half h = __float2half_rn((float)v);
        hi[d] = h;
        lo[d] = __float2half_rn((float)(v - (double)__half2float(h)));
    }
}

// The best L of n <= 512 scores (shared memory; slots `slot[i]`, or base + i), by one warp,
// written to out_s / out_i (slot -1 past the last), and the sums over the others (RegPart).
// The L-th largest of the 32 lane maxima bounds the L-th best score from below, so for
// L <= 32 only the few scores at or above it are collected and ranked by counting. More
// than 64 of them (ties), or a larger L, take L rounds of an arg-best over the warp.
__device__ __forceinline__ RegPart warp_select(const float* v, const int* slot, int base, int n, int L, float s2,
                               float* out_s, int* out_i, float* cs, int* ci) {
    const int lane = threadIdx.x & 31;
    constexpr unsigned full = 0xffffffffu;
    float a[16];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int e = lane + 32 * i;
        a[i] = e < n ? v[e] : -INFINITY;
        m = fmaxf(m, a[i]);
    }
    float ref = m;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ref = fmaxf(ref, __shfl_xor_sync(full, ref, o));
    uint32_t out_mask = 0;  // this lane's scores that went to the list
    float e0 = 0.0f, e1 = 0.0f;
    for (int j = lane; j < L; j += 32) {
        out_s[j] = -INFINITY;
        out_i[j] = -1;
    }
    __syncwarp();
    bool done = false;
    if (L <= 32) {
        int rank = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const float o = __shfl_sync(full, m, j);
            rank += (o > m || (o == m && j < lane)) ? 1 : 0;
        }
        const float tau =
            __shfl_sync(full, m, __ffs(__ballot_sync(full, rank == L - 1)) - 1);
        int cnt = 0;
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const bool in = a[i] >= tau && a[i] > -INFINITY;
            const unsigned b = __ballot_sync(full, in);
            const int pos = cnt + __popc(b & ((1u << lane) - 1));
            if (in && pos < 64) {
                const int e = lane + 32 * i;
                cs[pos] = a[i];
                ci[pos] = slot ? slot[e] : base + e;
            }
            mine |= in ? 1u << i : 0u;
            cnt += __popc(b);
        }
        __syncwarp();
        if (cnt <= 64) {
            out_mask = mine;
            done = true;
            for (int c = lane; c < cnt; c += 32) {
                const float s = cs[c];
                const int si = ci[c];
                int rk = 0;
                for (int j = 0; j < cnt; ++j) rk += ahead(cs[j], ci[j], s, si) ? 1 : 0;
                if (rk < L) {
                    out_s[rk] = s;
                    out_i[rk] = si;
                } else {
                    const float t = (s - ref) * s2, e = exp2f(t);
                    e0 += e;
                    e1 += e * t;
                }
            }
        }
    }
    if (!done) {
        for (int r = 0; r < L; ++r) {
            float bs = -INFINITY;
            int bi = INT_MAX, bp = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int e = lane + 32 * i;
                if (((out_mask >> i) & 1) || !(a[i] > -INFINITY)) continue;
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
                out_mask |= 1u << bp;
                out_s[r] = ws;
                out_i[r] = wi;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        // NaN scores (of a non-finite query) make the sums NaN; -inf adds nothing
        if (((out_mask >> i) & 1) || a[i] == -INFINITY) continue;
        const float t = (a[i] - ref) * s2, e = exp2f(t);
        e0 += e;
        e1 += e * t;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        e0 += __shfl_xor_sync(full, e0, o);
        e1 += __shfl_xor_sync(full, e1, o);
    }
    __syncwarp();
    return RegPart{ref, e0, e1};
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
};

// f64 cosine of a query with one slot, by one warp; `qq` gets |q|^2.
__device__ __forceinline__ double exact_cos(const MergeArgs& p, long long qrow, int slot, double& qq) {
    const int lane = threadIdx.x & 31;
    const uint8_t* codes = p.r.codes + slot * p.r.row_bytes;
    const uint8_t* group = p.r.group + (long long)slot * p.r.gpitch;
    double dot = 0.0, q2 = 0.0;
    int w2 = 0;
    for (int d0 = lane * 8; d0 < p.r.dim; d0 += 256) {
        int w[8];
        whole8(codes, group, p.r.bits, d0, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double v = d0 + j < p.r.dim ? (double)load_emb(p.q, p.q_type, qrow + d0 + j) : 0.0;
            dot += v * (double)w[j];
            q2 += v * v;
            w2 += w[j] * w[j];
        }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
        q2 += __shfl_xor_sync(0xffffffffu, q2, o);
    }
    w2 = __reduce_add_sync(0xffffffffu, w2);
    qq = q2;
    const double den = sqrt(q2) * sqrt((double)w2);
    return den > 0.0 ? dot / den : 0.0;
}

// Order-preserving map of a float to an unsigned key.
__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t b = __float_as_uint(f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}


// Exact cosines of the nb candidates `slots` and, as entry nb, of the query's label (slot 0
// stands in without one: the query's own length is wanted all the same), by all warps of
// the block. Returns the label's slot, -1 when there is none that is enrolled; *bad is set
// when the query holds an infinity or a NaN. The caller synchronises.
__device__ __forceinline__ int rescore(const MergeArgs& p, int qi, const int* slots, int nb,
                                       double* ex, int* bad) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int label = -1;
    if (p.labels) {
        label = p.labels[qi];
        if (label < 0 || label >= p.n_rows || !(p.r.scale[label] == p.r.scale[label])) label = -1;
    }
    for (int c = warp; c <= nb; c += blockDim.x / 32) {
        double qq;
        const double v = exact_cos(p, (long long)qi * p.ldq, c < nb ? slots[c] : max(label, 0), qq);
        if (lane == 0) {
            ex[c] = v;
            if (c == nb && !(qq <= 1.7976931348623157e308)) *bad = 1;
        }
    }
    return label;
}

// The best exact cosine M and its candidate (INT_MAX without any), by one warp.
__device__ __forceinline__ int find_top(const double* ex, int nb, double& M) {
    int at = INT_MAX;
    M = -INFINITY;
    for (int c = threadIdx.x & 31; c < nb; c += 32)
        if (ex[c] > M) M = ex[c], at = c;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const double om = __shfl_xor_sync(0xffffffffu, M, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (om > M || (om == M && oa < at)) M = om, at = oa;
    }
    return at;
}

// Writes a query's results, by one warp: E and S are the sums of e = exp(temperature (c - M))
// and of e temperature (c - M) over every score c but the top one.
__device__ __forceinline__ void write_posterior(const MergeArgs& p, int qi, const int* slots,
                                                const double* ex, int nb, bool bad, int label,
                                                double M, double E, double S) {
    const int lane = threadIdx.x & 31;
    const bool none = nb == 0;
    const double T = (double)p.temperature, lg = log1p(E);
    const float nan = __int_as_float(0x7FC00000);
    if (lane == 0) {
        p.lse[qi] = bad ? nan : none ? -INFINITY : (float)(T * M + lg);
        p.entropy[qi] = bad ? nan : none ? 0.0f : (float)(lg - S / (1.0 + E));
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
        int rank = 0;
        for (int j = 0; j < nb; ++j)
            rank += ahead((float)ex[j], slots[j], (float)ex[c], slots[c]) ? 1 : 0;
        if (rank < p.k) {
            p.alt_index[(long long)qi * p.k + rank] = slots[c];
            p.alt_log_prob[(long long)qi * p.k + rank] = (float)(T * (ex[c] - M) - lg);
        }
    }
}

// Largest dynamic shared memory each device has been asked to allow for one kernel.
struct SmemOptIn {
    std::mutex mu;
    size_t set[64] = {};
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
// Bytes of working memory, and the launches.
size_t registry_tc_work(int n_rows, int n_q, int dim, int k);
cudaError_t registry_tc_posterior(const MergeArgs& m, int k, void* work, cudaStream_t st);

}  // namespace vdb
