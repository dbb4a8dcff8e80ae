// Device helpers shared by the training kernels (q36moe_norm.hip,
// q36moe_rgrad.hip): row loads and stores in f32 or bf16, reductions over 16
// and 64 lanes, and the sum of partial rows.
#ifndef Q36MOE_ROWS_H
#define Q36MOE_ROWS_H
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "q36moe.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
// vectors at element alignment: rows of any width and stride start anywhere,
// and global loads and stores need no more than that
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_u __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

inline bool workspace_ok(const void *ws, size_t bytes, size_t need) {
    return need == 0 || (ws && bytes >= need && ((uintptr_t)ws & 15) == 0);
}

int hip_status(hipError_t e) { return e == hipSuccess ? Q36MOE_OK : Q36MOE_EHIP; }

__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
// two floats to bf16, round to nearest even (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// N consecutive elements (1, 4 or 8) of a row in format F, as floats.
template <int F, int N>
__device__ __forceinline__ void load_row(const void *p, size_t at, float (&v)[N]) {
    if constexpr (F == Q36MOE_FMT_F32) {
        const float *f = static_cast<const float *>(p) + at;
        if constexpr (N == 1) {
            v[0] = *f;
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const f32x4 t = *reinterpret_cast<const f32x4_u *>(f + i);
#pragma unroll
                for (int j = 0; j < 4; j++) v[i + j] = t[j];
            }
        }
    } else {
        const uint16_t *h = static_cast<const uint16_t *>(p) + at;
        if constexpr (N == 1) {
            v[0] = __uint_as_float((uint32_t)*h << 16);
        } else if constexpr (N == 4) {
            const u32x2_u t = *reinterpret_cast<const u32x2_u *>(h);
            v[0] = bf16_lo(t[0]); v[1] = bf16_hi(t[0]); v[2] = bf16_lo(t[1]); v[3] = bf16_hi(t[1]);
        } else {
            const u32x4_u t = *reinterpret_cast<const u32x4_u *>(h);
#pragma unroll
            for (int j = 0; j < 4; j++) { v[2 * j] = bf16_lo(t[j]); v[2 * j + 1] = bf16_hi(t[j]); }
        }
    }
}

// The same in two halves, for loads that are to be in flight while other work is
// done: the bits, and later their values.
template <int F, int N>
struct Bits {
    static constexpr int W = F == Q36MOE_FMT_F32 ? N : (N + 1) / 2;
    uint32_t u[W];
    __device__ __forceinline__ void load(const void *p, size_t at) {
        if constexpr (F == Q36MOE_FMT_F32) {
            const float *f = static_cast<const float *>(p) + at;
            if constexpr (N == 1) {
                u[0] = __float_as_uint(*f);
            } else {
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    const f32x4 t = *reinterpret_cast<const f32x4_u *>(f + i);
#pragma unroll
                    for (int j = 0; j < 4; j++) u[i + j] = __float_as_uint(t[j]);
                }
            }
        } else {
            const uint16_t *h = static_cast<const uint16_t *>(p) + at;
            if constexpr (N == 1) {
                u[0] = *h;
            } else if constexpr (N == 4) {
                const u32x2_u t = *reinterpret_cast<const u32x2_u *>(h);
                u[0] = t[0]; u[1] = t[1];
            } else {
                const u32x4_u t = *reinterpret_cast<const u32x4_u *>(h);
                u[0] = t[0]; u[1] = t[1]; u[2] = t[2]; u[3] = t[3];
            }
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (F == Q36MOE_FMT_F32) return __uint_as_float(u[i]);
        else return i & 1 ? bf16_hi(u[i / 2]) : bf16_lo(u[i / 2]);
    }
};

template <int F>
__device__ __forceinline__ void store_one(void *p, size_t at, float v) {
    if constexpr (F == Q36MOE_FMT_F32) static_cast<float *>(p)[at] = v;
    else static_cast<uint16_t *>(p)[at] = (uint16_t)bf16_pair(v, 0.0f);
}

// The elements from..N-1 of v to at.. (all of them in one or two stores).
template <int F, int N>
__device__ __forceinline__ void store_row(void *p, size_t at, const float (&v)[N], int from) {
    if (N == 1 || from) {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i >= from) store_one<F>(p, at + i, v[i]);
        return;
    }
    if constexpr (F == Q36MOE_FMT_F32) {
        float *f = static_cast<float *>(p) + at;
#pragma unroll
        for (int i = 0; i + 3 < N; i += 4) *reinterpret_cast<f32x4_u *>(f + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    } else {
        uint16_t *h = static_cast<uint16_t *>(p) + at;
        if constexpr (N == 4)
            *reinterpret_cast<u32x2_u *>(h) = u32x2_u{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
        else if constexpr (N == 8)
            *reinterpret_cast<u32x4_u *>(h) = u32x4_u{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]),
                                                      bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
    }
}

// Workgroup barrier for LDS data only: prefetched global loads stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

// Sum (maximum) over each row of 16 lanes, the same bits in all of them: quad
// xor 1, quad xor 2, half-row mirror, row mirror.
__device__ __forceinline__ float sum16(float v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    return v + dpp<0x140>(v);
}
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, dpp<0xB1>(v));
    v = fmaxf(v, dpp<0x4E>(v));
    v = fmaxf(v, dpp<0x141>(v));
    return fmaxf(v, dpp<0x140>(v));
}

// Sum over lanes l, l^16, l^32, l^48 (v_permlane16_swap / v_permlane32_swap put
// the halves side by side), and over the whole wave; all lanes get the same bits.
__device__ __forceinline__ float sum_rows4(float a) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(a), false, false);
    a = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(a), false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}
__device__ __forceinline__ float sum64(float v) { return sum_rows4(sum16(v)); }

// out[c] = sum over p < P of part[p * L + c]; columns from `split` on go to
// out2.  Many rows of few columns: a thread adds every 64th row of 4 columns, then
// the 64 sums of a column are added, in runs of 4 and those by a tree (512 rows of
// 3062 columns 4 us; 16 groups 12).  Few rows of many columns: 4 columns per
// thread, one row after the other (16 rows of 526336: 5 us, 6.5 TB/s; in groups
// as above 10).
__global__ __launch_bounds__(256) void k_sum_rows(const float *__restrict__ part, int P, size_t L, float *__restrict__ out) {
    const size_t c = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (c + 4 <= L) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 16
        for (int p = 0; p < P; p++) acc += *reinterpret_cast<const f32x4_u *>(part + (size_t)p * L + c);
        *reinterpret_cast<f32x4_u *>(out + c) = acc;
    } else {
        for (size_t o = c; o < L; o++) {
            float s = 0.0f;
            for (int p = 0; p < P; p++) s += part[(size_t)p * L + o];
            out[o] = s;
        }
    }
}

__global__ __launch_bounds__(256) void k_sum_partials(const float *__restrict__ part, int P, size_t L, size_t split,
                                                      float *__restrict__ out, float *__restrict__ out2) {
    constexpr int G = 64, C4 = 256 / G, C = 4 * C4;   // groups; columns per workgroup
    __shared__ __align__(16) float red[G][C];
    const int c4 = threadIdx.x % C4 * 4, g = threadIdx.x / C4;
    const size_t c = (size_t)blockIdx.x * C + c4;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (c + 4 <= L) {
#pragma unroll 8
        for (int p = g; p < P; p += G) acc += *reinterpret_cast<const f32x4_u *>(part + (size_t)p * L + c);
    } else {
        for (int p = g; p < P; p += G)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (c + i < L) acc[i] += part[(size_t)p * L + c + i];
    }
    *reinterpret_cast<f32x4 *>(&red[g][c4]) = acc;
    __syncthreads();
    const int col = threadIdx.x >> 4, l = threadIdx.x & 15;   // 16 lanes per column
    float s = red[4 * l][col];
#pragma unroll
    for (int i = 1; i < 4; i++) s += red[4 * l + i][col];
    s = sum16(s);
    const size_t o = (size_t)blockIdx.x * C + col;
    if (l == 0) {
        if (o < split) out[o] = s;
        else if (o < L) out2[o - split] = s;
    }
}

inline void sum_partials(const float *part, int P, size_t L, size_t split, float *out, float *out2, hipStream_t s) {
    if (P <= 32 && L > 65536 && split == L)
        hipLaunchKernelGGL(k_sum_rows, dim3((unsigned)((L + 1023) / 1024)), dim3(256), 0, s, part, P, L, out);
    else
        hipLaunchKernelGGL(k_sum_partials, dim3((unsigned)((L + 15) / 16)), dim3(256), 0, s, part, P, L, split, out, out2);
}

}  // namespace
#endif
