// Shared pieces of the quantised speaker registry's kernels (registry.cu,
// registry_tc.cu): the row layout, loads of the embedding types, the softmax partials and
// the candidate order. See vdb_ops.h for the stored format.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

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

template <int T>
struct EmbType;
template <>
struct EmbType<kF32> {
    using type = float;
};
template <>
struct EmbType<kF16> {
    using type = __half;
};
template <>
struct EmbType<kBF16> {
    using type = __nv_bfloat16;
};

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

// Whole number of dimension d of a row (codes and group scales of that row).
__device__ __forceinline__ int reg_whole(const uint8_t* codes, const uint8_t* group, int bits,
                                         int d) {
    if (bits == 8) return (int)codes[d] - 128;
    const int j = d & 7, n = (j >> 1) + (j & 1) * 4;  // nibble of the word
    const int byte = (d & ~7) / 2 + (n >> 1);
    return (((int)codes[byte] >> ((n & 1) * 4) & 15) - 8) * (int)group[d >> 5];
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

}  // namespace vdb
