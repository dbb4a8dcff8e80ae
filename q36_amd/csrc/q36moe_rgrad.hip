// Training the router: per-expert counts and the balance loss, the gradient of
// the router logits, and the gradients of the router product.
//
//   p_t = softmax(logits_t),  c_e picks of expert e and P_e = sum_t p_te over
//   the n live tokens,  f_e = c_e / (n k):
//   balance loss        coef * E * sum_e f_e P_e / n
//   its gradient        dlogits_t = dloss * coef * E / n * p_t * (f - <p_t, f>)
//   routing weights     q = softmax over a token's picks, wt = scale * q:
//                       dlogits_s = scale * q_s * (dwt_s - <q, dwt>)
//   (not renormalised)  u_e = scale * sum of dwt_s over picks of e:
//                       dlogits = p * (u - <p, u>)
//   router product      dW = dlogits^T x,  dx = dlogits W
#include "q36moe_rows.h"

#include <type_traits>

namespace {

constexpr int kMaxE = 256, kMaxK = 8;

// A wave's LDS writes before its reads.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A token's E values in 16 lanes: lane l holds columns 64 i + 4 l..+3 in v[i],
// so that rows move as 16-byte vectors where E is a multiple of 4 (whatever
// their alignment) and as single values elsewhere.  Columns past E read as
// `fill`.
template <int NV>
__device__ __forceinline__ void load16(const float *__restrict__ row, int E, int l, float fill, float (&v)[NV][4]) {
    if ((E & 3) == 0) {
#pragma unroll
        for (int i = 0; i < NV; i++) load_row<Q36MOE_FMT_F32>(row, min(64 * i + 4 * l, E - 4), v[i]);
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) v[i][c] = 64 * i + 4 * l < E ? v[i][c] : fill;
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) v[i][c] = row[min(64 * i + 4 * l + c, E - 1)];
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) v[i][c] = 64 * i + 4 * l + c < E ? v[i][c] : fill;
    }
}

template <int NV>
__device__ __forceinline__ void store16(float *__restrict__ row, int E, int l, const float (&v)[NV][4]) {
    if ((E & 3) == 0) {
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (64 * i + 4 * l < E) store_row<Q36MOE_FMT_F32>(row, 64 * i + 4 * l, v[i], 0);
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (64 * i + 4 * l + c < E) row[64 * i + 4 * l + c] = v[i][c];
    }
}

// Softmax of the values that 16 lanes hold: v becomes exp(v - max), and one over
// their sum is returned; a row of -inf has no probabilities, all 0.  Two roundings
// of the exponent, 2^-23 |v - max| of the value.
template <int NV, int NC>
__device__ __forceinline__ float softmax16(float (&v)[NV][NC]) {
    constexpr float kLog2e = 1.44269504088896341f;
    float m = v[0][0];
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int c = 0; c < NC; c++) m = fmaxf(m, v[i][c]);
    m = max16(m);
    m = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int c = 0; c < NC; c++) {
            v[i][c] = __builtin_amdgcn_exp2f((v[i][c] - m) * kLog2e);
            s += v[i][c];
        }
    s = sum16(s);
    return s == 0.0f ? 0.0f : 1.0f / s;   // a NaN stays one
}

template <int NV>
__device__ __forceinline__ float dot16(const float (&a)[NV][4], const float (&b)[NV][4]) {
    float d = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) d = fmaf(a[i][c], b[i][c], d);
    return sum16(d);
}

// ---------------------------------------------------------------------------
// counts, summed probabilities, balance loss
// ---------------------------------------------------------------------------
struct BalanceArgs {
    const float *logits;
    const int32_t *idx;
    const uint8_t *mask;
    int ld, T, E, k, chunk;    // tokens per workgroup
    float coef;
    int32_t *counts;           // [E + 1]
    float *psum, *loss;        // [E], [1]
    // of more than one workgroup: [workgroups][E + 1] sum of probabilities and
    // count, then a partial loss per joining workgroup, live tokens, arrivals
    float2 *part;
};

constexpr int kBalW = 16;                        // waves per workgroup
constexpr int kBalGroups = 256;                  // most workgroups
constexpr int kJoinE = 16;                       // counters per joining workgroup
constexpr int kJoins = (kMaxE + 1 + kJoinE - 1) / kJoinE;
struct BalanceJoin {
    double loss[kJoins];
    int32_t live, arrived;
};
__host__ __device__ inline size_t balance_part_bytes(int nb, int E) { return ((size_t)nb * (E + 1) * sizeof(float2) + 15) / 16 * 16; }

// coef * E / (k n^2) times the sum of counts times sums of probabilities, which
// is formed in 64 bits.
__device__ __forceinline__ float balance_of(const BalanceArgs &A, double s, int32_t live) {
    const double n = (double)live;
    return live > 0 ? (float)((double)A.coef * A.E * s / ((double)A.k * n * n)) : 0.0f;
}

// 16 lanes per token, 64 tokens of the workgroup's run at a time, the next
// token's loads ahead of the sums of this one.  What bounds a workgroup is the
// vector unit: 64 tokens of 256 experts take a CU 1.4 us, so the tokens are spread
// over all of them.
template <int NV>
__global__ __launch_bounds__(64 * kBalW) void k_balance(BalanceArgs A) {
    __shared__ __align__(16) float ps[kBalW][64 * NV];
    __shared__ int32_t cnt[kMaxE + 1];
    const int tid = threadIdx.x, l = tid & 15, wave = tid >> 6;
    const int64_t t0 = (int64_t)blockIdx.x * A.chunk, t1 = min(t0 + A.chunk, (int64_t)A.T);
    if (gridDim.x > 1 && blockIdx.x == 0 && tid == 0)   // for the joining kernel, which runs after this one
        reinterpret_cast<BalanceJoin *>(reinterpret_cast<uint8_t *>(A.part) + balance_part_bytes(gridDim.x, A.E))->arrived = 0;
    for (int e = tid; e <= A.E; e += 64 * kBalW) cnt[e] = 0;
    __syncthreads();
    float acc[NV][4] = {}, v[NV][4];
    int pick = -1, n = 0;
    bool live = false;
    auto load = [&](int64_t t) {
        live = t < t1;
        const int64_t tc = min(t, t1 - 1);   // a run without tokens has no logits to read
        if (tc >= t0) {
            load16(A.logits + (size_t)tc * A.ld, A.E, l, -INFINITY, v);
            pick = l < A.k ? A.idx[(size_t)tc * A.k + l] : -1;
            if (A.mask) live = live && A.mask[tc];
        }
    };
    int64_t t = t0 + (tid >> 4);
    load(t);
    for (; t < t1; t += 4 * kBalW) {
        float p[NV][4];
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) p[i][c] = v[i][c];
        const bool counted = live;
        if (counted) {
            if ((unsigned)pick < (unsigned)A.E) atomicAdd(&cnt[pick], 1);
            n += l == 0;
        }
        load(t + 4 * kBalW);
        const float inv = softmax16(p);
        if (counted)   // padding may hold anything
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) acc[i][c] = fmaf(p[i][c], inv, acc[i][c]);
    }
    if (n) atomicAdd(&cnt[A.E], n);
#pragma unroll
    for (int i = 0; i < NV; i++) {
#pragma unroll
        for (int c = 0; c < 4; c++) acc[i][c] = sum_rows4(acc[i][c]);
        if ((tid & 63) < 16) *reinterpret_cast<float4 *>(&ps[wave][64 * i + 4 * l]) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    }
    __syncthreads();
    float s = 0.0f;
    const int e = tid;
    if (e < A.E) {
        s = ps[0][e];
#pragma unroll
        for (int w = 1; w < kBalW; w++) s += ps[w][e];
    }
    if (gridDim.x > 1) {
        if (e <= A.E) A.part[(size_t)blockIdx.x * (A.E + 1) + e] = make_float2(s, __int_as_float(cnt[e]));
        return;
    }
    __syncthreads();
    if (e < A.E) {
        A.psum[e] = s;
        ps[0][e] = s;
    }
    if (e <= A.E) A.counts[e] = cnt[e];
    __syncthreads();
    if (wave == 0) {
        double d = 0.0;
#pragma unroll
        for (int i = 0; i < kMaxE / 64; i++)
            if (tid + 64 * i < A.E) d += (double)cnt[tid + 64 * i] * (double)ps[0][tid + 64 * i];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
        if (tid == 0) *A.loss = balance_of(A, d, cnt[A.E]);
    }
}

// The workgroups' parts to counts, sums and loss, 16 counters per workgroup (one
// CU alone brings 50 GB/s in: 128 parts took it 6.8 us).  The workgroup that
// arrives last adds the partial losses, in the order of the experts.
__global__ __launch_bounds__(256) void k_balance_join(BalanceArgs A, int nb) {
    __shared__ float ps[16][kJoinE];
    __shared__ int32_t cs[16][kJoinE];
    __shared__ int last;
    BalanceJoin *J = reinterpret_cast<BalanceJoin *>(reinterpret_cast<uint8_t *>(A.part) + balance_part_bytes(nb, A.E));
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4, e = blockIdx.x * kJoinE + c, n = A.E + 1;
    float s = 0.0f;
    int32_t k = 0;
    if (e < n)
#pragma unroll 16
        for (int b = g; b < nb; b += 16) {
            const float2 v = A.part[(size_t)b * n + e];
            s += v.x;
            k += __float_as_int(v.y);
        }
    ps[g][c] = s;
    cs[g][c] = k;
    __syncthreads();
    if (threadIdx.x < kJoinE) {
        s = 0.0f;
        k = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            s += ps[i][c];
            k += cs[i][c];
        }
        if (e < n) A.counts[e] = k;
        if (e < A.E) A.psum[e] = s;
        double d = e < A.E ? (double)k * (double)s : 0.0;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) d += __shfl_xor(d, o, 16);
        if (e == A.E) __hip_atomic_store(&J->live, k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (c == 0) __hip_atomic_store(&J->loss[blockIdx.x], d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __threadfence();
        if (c == 0) last = __hip_atomic_fetch_add(&J->arrived, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (threadIdx.x == 0 && last) {
        __threadfence();
        double d = 0.0;
        for (int b = 0; b < (int)gridDim.x; b++) d += __hip_atomic_load(&J->loss[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *A.loss = balance_of(A, d, __hip_atomic_load(&J->live, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    }
}

// Workgroups: one up to 384 tokens, which saves the second launch and the
// workspace, then one per 64 tokens, and from 16384 tokens on one per CU.  us on the
// GPU, one workgroup / more: 256 tokens 9.6 / 11.1, 400 12.6 / 11.3, 600 16.8 / 11.2;
// at 32768 tokens 64 / 128 / 256 workgroups 23.1 / 18.3 / 14.6.
int balance_groups(int T) {
    if (T <= 384) return 1;
    const int n = (int)(((int64_t)T + 63) / 64);
    return n < kBalGroups ? n : kBalGroups;
}

// ---------------------------------------------------------------------------
// gradient of the logits
// ---------------------------------------------------------------------------
struct LogitGradArgs {
    const float *logits;
    const int32_t *idx;
    const float *dwt;
    const int32_t *counts;
    const uint8_t *mask;
    const float *dloss;
    float *out;
    int ld, ldo, T, E, k, renorm;
    float scale, coef;
};

// 16 lanes per token, 16 tokens per workgroup.  FULL: the softmax over all
// experts, for the balance loss or for weights that are not renormalised; without
// it a token's logits are read at its picks alone.  Lane s < k forms the gradient
// of pick s and puts it into the token's row in LDS, from where the lanes that
// hold its expert take it; where an expert stands twice the picks are added one
// after the other instead, in slot order.  Both parts for 16384 tokens of 256
// experts 12 us (2.9 TB/s); comparing every pick with every expert in registers took
// 19, single loads instead of 16-byte vectors and all.
template <int NV, bool FULL>
__global__ __launch_bounds__(256) void k_logit_grad(LogitGradArgs A) {
    constexpr int LDS = 64 * NV + 16;   // floats per row: the four tokens of a wave 16 banks apart
    __shared__ __align__(16) float up_row[16][LDS];
    const int l = threadIdx.x & 15, slot = threadIdx.x >> 4;
    const bool balance = FULL && A.counts;
    float f[NV][4];
    float gain = 0.0f;
    if (balance) {
        const float n = (float)A.counts[A.E];
        const float inv = n > 0.0f ? 1.0f / (n * (float)A.k) : 0.0f;
        gain = n > 0.0f ? A.coef * (float)A.E / n * (A.dloss ? *A.dloss : 1.0f) : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) f[i][c] = (float)A.counts[min(64 * i + 4 * l + c, A.E - 1)] * inv;
    }
    for (int64_t t = (int64_t)blockIdx.x * 16 + slot; t < A.T; t += (int64_t)gridDim.x * 16) {
        const float *row = A.logits + (size_t)t * A.ld;
        const bool live = !A.mask || A.mask[t];
        float p[NV][4], u[NV][4];
        int e = -1;
        float up = 0.0f, lp = -INFINITY;
        if (A.dwt && l < A.k) {
            e = A.idx[(size_t)t * A.k + l];
            up = A.dwt[(size_t)t * A.k + l] * A.scale;
            e = (unsigned)e < (unsigned)A.E ? e : -1;   // an index that names no expert: no pick
        }
        if (FULL) load16(row, A.E, l, -INFINITY, p);
        if (A.dwt) {
            if (A.renorm && e >= 0) lp = row[e];
            float s = e >= 0 ? up : 0.0f;
            if (A.renorm) {
                float q[1][1] = {{lp}};
                const float share = softmax16(q) * q[0][0];
                const float mean = sum16(share * s);   // by all 16 lanes, those without a pick too
                s = e >= 0 ? share * (up - mean) : 0.0f;
            }
            // the same expert at two slots of a token: compared with the lanes
            // 1..7 to the right in the row
            bool twice = false;
#define SAME(N) twice |= __builtin_amdgcn_update_dpp(-2, e, 0x100 + N, 0xf, 0xf, false) == e
            SAME(1); SAME(2); SAME(3); SAME(4); SAME(5); SAME(6); SAME(7);
#undef SAME
            twice = twice && e >= 0;
            float *mine = up_row[slot];
#pragma unroll
            for (int i = 0; i < NV; i++) *reinterpret_cast<float4 *>(&mine[64 * i + 4 * l]) = make_float4(0.f, 0.f, 0.f, 0.f);
            wave_sync();
            if (!__any(twice)) {
                if (e >= 0) mine[e] = s;
            } else {
                for (int j = 0; j < kMaxK; j++) {
                    if (l == j && e >= 0) mine[e] += s;
                    wave_sync();
                }
            }
            wave_sync();
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const float4 v = *reinterpret_cast<const float4 *>(&mine[64 * i + 4 * l]);
                u[i][0] = v.x; u[i][1] = v.y; u[i][2] = v.z; u[i][3] = v.w;
            }
            wave_sync();
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) u[i][c] = 0.0f;
        }
        if (FULL) {
            const float inv = softmax16(p);
            const float d = balance ? dot16(p, f) * inv : 0.0f;
            const float du = A.dwt && !A.renorm ? dot16(p, u) * inv : 0.0f;
            const float gi = gain * inv;
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    if (!A.renorm) u[i][c] = p[i][c] * inv * (u[i][c] - du);
                    if (balance) u[i][c] = fmaf(gi * p[i][c], f[i][c] - d, u[i][c]);
                }
        }
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) u[i][c] = live ? u[i][c] : 0.0f;
        store16(A.out + (size_t)t * A.ldo, A.E, l, u);
    }
}

// ---------------------------------------------------------------------------
// gradients of the router product
// ---------------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

constexpr int kRgD = 2048;
constexpr int kMaxRouterT = 1 << 23, kMaxRouterRows = 1 << 20, kMaxRouterLd = 1 << 22;

struct ProductArgs {
    const float *w, *dl, *dsh;   // [n_rows][kRgD]; [T][ld]; the shared gate's column, stride ld_sh
    const void *x;
    float *dw;                   // [splits][n_rows][kRgD]
    void *dx;
    int ld, ld_sh, n_rows, n_expert, T;
    int span;                    // split dW: tokens per split
    int parts;                   // dx on f16: workgroups that share the columns of 256 tokens
    int nw;                      // fp32: workgroups of dW in front of those of dx
};

// Row of C's register i: all three MFMAs of 32 x 32 hold rows 8 (i / 4) +
// 4 (L / 32) + i % 4 of column L % 32 in lane L.
__device__ __forceinline__ int c_row(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }


// Workgroup b of n in an order in which those of one XCD (b % 8) are neighbours.
__device__ __forceinline__ int xcd_order(int b, int n) { return (n & 7) ? b : (b & 7) * (n >> 3) + (b >> 3); }

// ---- few tokens: fp32 MFMA ----
// v_mfma_f32_32x32x2_f32: lane L holds row (A) or column (B) L % 32 at K element
// L / 32.  One tile of 32 rows x 64 columns per workgroup, whose four waves take a
// quarter of K each and add up through LDS: at these sizes a tile's time is the
// round trips of its loads (203 tokens, a wave per 32 x 32 tile and all of K: dW
// 10.6, dx 9.4 us).  Operands come straight from the caches in batches, the next
// batch's loads ahead of the products of this one.  dW and dx share the launch.
constexpr int kF32Cols = 64;

template <int XF>
__device__ __forceinline__ float load_x(const void *x, size_t at) {
    if constexpr (XF == Q36MOE_FMT_F32) return static_cast<const float *>(x)[at];
    else return __uint_as_float((uint32_t)static_cast<const uint16_t *>(x)[at] << 16);
}

struct Tile2 { f32x16 c[2]; };   // columns L % 32 and 32 + L % 32

__device__ __forceinline__ void mfma2(Tile2 &t, float a, float b0, float b1) {
    t.c[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b0, t.c[0], 0, 0, 0);
    t.c[1] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b1, t.c[1], 0, 0, 0);
}

// A quarter of the tokens: dlogits^T x.  Batches of 16 K-steps; tokens past the
// end read the last one and count as zeros.
template <int XF>
__device__ __forceinline__ Tile2 f32_dw_dot(const ProductArgs &A, int wave, int half, const float *col, int64_t step, int d) {
    constexpr int U = 16;
    Tile2 acc = {};
    const int quarter = ((A.T + 7) >> 3) << 1, t0 = wave * quarter, t1 = min(t0 + quarter, A.T);
    float a[2][U], b[2][U][2];
    auto load = [&](int t, float (&av)[U], float (&bv)[U][2]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int tc = min(t + 2 * u + half, t1 - 1);
            av[u] = col[tc * step];
            bv[u][0] = load_x<XF>(A.x, (size_t)tc * kRgD + d);
            bv[u][1] = load_x<XF>(A.x, (size_t)tc * kRgD + d + 32);
        }
    };
    auto products = [&](int t, const float (&av)[U], const float (&bv)[U][2]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool in = t + 2 * u + half < t1;
            mfma2(acc, in ? av[u] : 0.0f, in ? bv[u][0] : 0.0f, in ? bv[u][1] : 0.0f);
        }
    };
    if (t0 >= t1) return acc;
    load(t0, a[0], b[0]);
    for (int t = t0; t < t1; t += 4 * U) {
        if (t + 2 * U < t1) load(t + 2 * U, a[1], b[1]);
        products(t, a[0], b[0]);
        if (t + 2 * U < t1) {
            if (t + 4 * U < t1) load(t + 4 * U, a[0], b[0]);
            products(t + 2 * U, a[1], b[1]);
        }
    }
    return acc;
}

// A quarter of a token's router rows: dlogits W.  The rows are neighbours in
// memory, so a lane takes four at a time (half h of a step of 8 holds rows
// 4 h..4 h + 3 of both operands; one row per load, with 64 lanes in 32 tokens'
// rows, nearly doubled the time).  The rows past the last whole step, the shared
// gate's among them, go to the last wave.
__device__ __forceinline__ Tile2 f32_dx_dot(const ProductArgs &A, int wave, int half, const float *row, const float *gate,
                                            const float *col) {
    constexpr int U = 4;
    Tile2 acc = {};
    float a[2][U][4], b[2][U][4][2];
    const int whole = A.n_expert & ~7, quarter = ((whole >> 3) + 3) / 4 * 8;
    const int k0 = wave * quarter, k1 = min(k0 + quarter, whole);
    auto load = [&](int k, float (&av)[U][4], float (&bv)[U][4][2]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = min(k + 8 * u, k1 - 8) + 4 * half;   // past the end the last step again
            load_row<Q36MOE_FMT_F32>(row, r, av[u]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                bv[u][i][0] = col[(size_t)(r + i) * kRgD];
                bv[u][i][1] = col[(size_t)(r + i) * kRgD + 32];
            }
        }
    };
    auto products = [&](int k, const float (&av)[U][4], const float (&bv)[U][4][2]) {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (k + 8 * u < k1)
#pragma unroll
                for (int i = 0; i < 4; i++) mfma2(acc, av[u][i], bv[u][i][0], bv[u][i][1]);
    };
    if (k0 < k1) {
        load(k0, a[0], b[0]);
        for (int k = k0; k < k1; k += 16 * U) {
            if (k + 8 * U < k1) load(k + 8 * U, a[1], b[1]);
            products(k, a[0], b[0]);
            if (k + 8 * U < k1) {
                if (k + 16 * U < k1) load(k + 16 * U, a[0], b[0]);
                products(k + 8 * U, a[1], b[1]);
            }
        }
    }
    if (wave == 3 && whole < A.n_rows) {
        float av[4], b0[4], b1[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int r = min(whole + 2 * u + half, A.n_rows - 1);
            av[u] = r < A.n_expert ? row[r] : *gate;
            b0[u] = col[(size_t)r * kRgD];
            b1[u] = col[(size_t)r * kRgD + 32];
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const bool in = whole + 2 * u + half < A.n_rows;
            mfma2(acc, in ? av[u] : 0.0f, in ? b0[u] : 0.0f, in ? b1[u] : 0.0f);
        }
    }
    return acc;
}

template <int XF>
__global__ __launch_bounds__(256) void k_router_grad_f32(ProductArgs A) {
    __shared__ float red[4][32][64];
    const int lane = threadIdx.x & 63, half = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool is_dw = (int)blockIdx.x < A.nw;
    const int b = is_dw ? blockIdx.x : blockIdx.x - A.nw;
    const int d = b % (kRgD / kF32Cols) * kF32Cols + c, m0 = b / (kRgD / kF32Cols) * 32;
    Tile2 acc;
    if (is_dw) {
        const int r = min(m0 + c, A.n_rows - 1);
        const bool sh = r >= A.n_expert;
        acc = f32_dw_dot<XF>(A, wave, half, sh ? A.dsh : A.dl + r, sh ? A.ld_sh : A.ld, d);
    } else {
        const int t = min(m0 + c, A.T - 1);
        acc = f32_dx_dot(A, wave, half, A.dl + (size_t)t * A.ld, A.dsh + (int64_t)t * A.ld_sh, A.w + d);
    }
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < 16; i++) red[wave][16 * j + i][lane] = acc.c[j][i];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 8; q++) {
        const int i = 8 * wave + q, m = m0 + c_row(i & 15, lane), col = d + 32 * (i >> 4);
        const float v = (red[0][i][lane] + red[1][i][lane]) + (red[2][i][lane] + red[3][i][lane]);
        if (is_dw) {
            if (m < A.n_rows) A.dw[(size_t)m * kRgD + col] = v;
        } else if (m < A.T) {
            store_one<XF>(A.dx, (size_t)m * kRgD + col, v);
        }
    }
}

// ---- many tokens: operands split into f16 ----
// v_mfma_f32_32x32x16_f16 takes 32 cycles for eight times the products of the
// fp32 MFMA.  An fp32 value times a power of two that puts the largest of its row
// or column near the top of f16's range is the sum of two f16 (11 bits each) to
// 2^-22 of itself, or to 2^-25 of the scaled range's unit where that is more; three
// of the four products of two such sums give fp32's exactness (the fourth is 2^-22
// of the first).  A bf16 value is one f16.  Products of three bf16 pieces need no
// scaling but are six (three with bf16 x): with random operands the chip holds
// about 1200 TFLOP/s, and dW of 16384 tokens took 93 us with them (58 bf16).
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Exponent e <= 126 (so that 2^e is a float) with amax * 2^e in [2^top, 2^(top+1)),
// for inf and NaN as if they were 2^128.
__device__ __forceinline__ int scale_exp(float amax, int top) {
    return min(top + 127 - (int)(__float_as_uint(amax) >> 23), 126);
}

// v * scale as NP f16 pieces.
template <int NP>
__device__ __forceinline__ void split_f16(const float (&v)[8], float scale, f16x8 (&p)[NP]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float s = v[i] * scale;
        p[0][i] = (_Float16)s;
        if constexpr (NP > 1) p[1][i] = (_Float16)(s - (float)p[0][i]);
    }
}

// ---- dW ----
// Workgroup: 32 MW router rows x 128 columns over the tokens of its split, 8
// waves as MW x 8 / MW.  Lane L of an operand holds row (column) L % 32 at K
// elements (tokens) 8 (L / 32)..+7.  A wave reads its rows of the logits'
// gradient straight into that order (32 neighbouring values per load) and splits
// them itself; x is split once per workgroup and shared through LDS in operand
// order, two buffers, one barrier per 64 tokens.  The columns of MFMA tiles 2q
// and 2q + 1 interleave, so pairs of columns load and store as 8 bytes.
// The shared gate's row is an fp32 sum beside the conversion of x.
//   Scales: a row's (column's) is chosen from its first 64 tokens, whose largest
// value it puts at 2^10..2^11, and lowered, the sums so far with it, when a later
// value would pass f16's largest: looked for in each step's loads a step before
// their use, by a wave alone in its rows, and in the columns by a flag that the
// workgroup sees behind the barrier.  The sums follow after the products of the
// values that still had the old scale.
//   4096 / 16384 fp32 tokens and 256 rows 33 / 73 us with the sum of the splits
// (bf16 x 28 / 55).  The splits' parts, 33.5 MB at 256 rows, are one tile per CU.
constexpr int kDwCols = 128, kDwStep = 64, kDwTop = 10;
constexpr float kF16Max = 65504.0f;

template <int XF, int MW>
__global__ __launch_bounds__(512) void k_router_dw_split(ProductArgs A) {
    constexpr bool F32 = XF == Q36MOE_FMT_F32;
    constexpr int NP = F32 ? 2 : 1;           // pieces of x
    constexpr int NT = MW / 2;                // tiles per wave
    __shared__ __align__(16) f16x8 sx[2][NP][4][4][64];
    __shared__ float scol[8][kDwCols];        // columns' maxima, and the gate's sums at the end
    __shared__ int ecol[kDwCols], shift[kDwCols];
    // per x buffer, as a wave may end a step, and set the next one's, while another
    // has yet to read this one's
    __shared__ int flag[2];
    const int lane = threadIdx.x & 63, half = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % MW, wn = wave / MW;
    const int mblocks = (A.n_expert + 32 * MW - 1) / (32 * MW), tiles = kRgD / kDwCols * mblocks;
    const int b = xcd_order(blockIdx.x, gridDim.x);
    const int split = b / tiles, n0 = b % tiles % (kRgD / kDwCols) * kDwCols, mb = b % tiles / (kRgD / kDwCols);
    const int r0 = (mb * MW + wm) * 32;
    const int t0 = split * A.span, t1 = min(t0 + A.span, A.T);
    const bool gate = A.n_rows > A.n_expert && mb == 0;
    // the shared gate's gradients, or any others where no row of it is formed
    // (its sums are then not stored): no condition in the loop
    const float *gcol = gate ? A.dsh : A.dl;
    const int64_t gstep = gate ? A.ld_sh : A.ld;

    f32x16 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j] = f32x16{};
    float sg[2] = {0.0f, 0.0f};
    float a[2][4][8];
    uint32_t xr[8][F32 ? 2 : 1];              // tokens t + 8 wave + i, columns n0 + 2 lane, + 1
    float sh;                                 // the gate's gradient of token t + 8 wave + lane % 8
    int er, ex[2];                            // exponents of the lane's row and of its columns of x

    // Whole steps load through buffers based at the step's first row, with the
    // rows as scalar offsets: no address arithmetic on the vector unit.  In the
    // split's last step tokens past its end are zeros.
    const int lr = min(r0 + c, A.n_expert - 1);
    const uint32_t lo = (uint32_t)(8 * half * A.ld + lr) * 4u;
    auto load_x = [&](int t, auto WHOLE) {
        const int tx = t + 8 * wave;
        if (decltype(WHOLE)::value || t + kDwStep <= t1) {
            const size_t at = (size_t)tx * kRgD + n0;
            if constexpr (F32) {
                const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                    const_cast<float *>(static_cast<const float *>(A.x) + at), (short)0, 0x7ffffffe, 0x00020000);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, lane * 8, i * kRgD * 4, 0);
                    xr[i][0] = v[0];
                    xr[i][1] = v[1];
                }
            } else {
                const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                    const_cast<uint16_t *>(static_cast<const uint16_t *>(A.x) + at), (short)0, 0x7ffffffe, 0x00020000);
#pragma unroll
                for (int i = 0; i < 8; i++) xr[i][0] = __builtin_amdgcn_raw_buffer_load_b32(r, lane * 4, i * kRgD * 2, 0);
            }
            sh = gcol[(tx + (lane & 7)) * gstep];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int tc = min(tx + i, t1 - 1);
                const size_t at = (size_t)tc * kRgD + n0 + 2 * lane;
                uint32_t v0, v1 = 0;
                if constexpr (F32) {
                    v0 = static_cast<const uint32_t *>(A.x)[at];
                    v1 = static_cast<const uint32_t *>(A.x)[at + 1];
                } else {
                    v0 = *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(A.x) + at);
                }
                xr[i][0] = tx + i < t1 ? v0 : 0u;
                if constexpr (F32) xr[i][1] = tx + i < t1 ? v1 : 0u;
            }
            const float v = gcol[min(tx + (lane & 7), t1 - 1) * gstep];
            sh = tx + (lane & 7) < t1 ? v : 0.0f;
        }
    };
    auto x_at = [&](int i, int u) {
        return F32 ? __uint_as_float(xr[i][F32 ? u : 0]) : u ? bf16_hi(xr[i][0]) : bf16_lo(xr[i][0]);
    };
    auto load_a = [&](int t, float (&av)[4][8], auto WHOLE) {
        if (decltype(WHOLE)::value || t + kDwStep <= t1) {
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(A.dl + (size_t)t * A.ld), (short)0,
                                                                               0x7ffffffe, 0x00020000);
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    av[k][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, lo, (16 * k + i) * A.ld * 4, 0));
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int tt = t + 16 * k + 8 * half + i;
                    const float v = A.dl[(size_t)min(tt, t1 - 1) * A.ld + lr];
                    av[k][i] = tt < t1 ? v : 0.0f;
                }
        }
    };
    auto row_max = [&](const float (&av)[4][8]) {
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(av[k][i]));
        return m;
    };
    // the wave's tokens of x to LDS and to the shared gate's sums
    auto convert = [&](int buf) {
        const int k = wave >> 1, at = (lane & 31) + 32 * (wave & 1), q = lane >> 5;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = x_at(i, u);
            f16x8 p[NP];
            split_f16<NP>(v, pow2(ex[u]), p);
#pragma unroll
            for (int n = 0; n < NP; n++) sx[buf][n][k][2 * q + u][at] = p[n];
#pragma unroll
            for (int i = 0; i < 8; i++) sg[u] = fmaf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(sh), i)), v[i], sg[u]);
        }
    };
    auto x_max = [&](float (&m)[2]) {
        m[0] = m[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int u = 0; u < 2; u++) m[u] = fmaxf(m[u], fabsf(x_at(i, u)));
    };
    auto check_x = [&](int buf) {             // does the step in xr fit its scales? asked in the step of buf
        float m[2];
        x_max(m);
        if (m[0] * pow2(ex[0]) > kF16Max || m[1] * pow2(ex[1]) > kF16Max) flag[buf] = 1;
    };
    // the scales of x for the step in xr, lowered where they do not fit (FIRST:
    // chosen); shift[] holds by how much.  Ends with a barrier.
    auto fit_x = [&](int buf, auto FIRST) {
        float m[2];
        x_max(m);
        *reinterpret_cast<float2 *>(&scol[wave][2 * lane]) = make_float2(m[0], m[1]);
        lds_barrier();
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float all = scol[0][2 * lane + u];
#pragma unroll
            for (int k = 1; k < 8; k++) all = fmaxf(all, scol[k][2 * lane + u]);
            const int old = ex[u];
            if (decltype(FIRST)::value || all * pow2(old) > kF16Max) ex[u] = scale_exp(all, kDwTop);
            if (wave == 0) {
                ecol[2 * lane + u] = ex[u];
                shift[2 * lane + u] = decltype(FIRST)::value ? 0 : ex[u] - old;
            }
        }
        if (wave == 0) {
            flag[buf] = 0;
            if (decltype(FIRST)::value) flag[buf ^ 1] = 0;
        }
        lds_barrier();
    };
    auto col_of = [&](int j) { const int q = wn * NT + j; return 64 * (q >> 1) + 2 * c + (q & 1); };

    // One step: the products of its 64 tokens from LDS, and beside them, in the
    // 32 cycles that each MFMA runs, the split of the next 16 tokens' gradients,
    // the conversion of the next step's x into the other buffer and the loads of
    // the step after it.  One barrier: a step's x is in LDS before it, and every
    // wave has read the buffer that is written after it.  The steady steps have
    // no conditions, which keeps them one block for the scheduler and the waits
    // before a use counted (after a load that may not have been made they are for
    // every load).
    f16x8 s[2];                               // of this step's first 16 tokens
    constexpr int NM = NP + 1;                // products per tile and 16 tokens
    // the order of a block of K x 16 tokens: LDS reads of a tile (with bf16 x, whose
    // registers allow it, a tile ahead), then its MFMAs with V vector instructions
    // behind each (masks: 0x100 LDS read, 0x8 MFMA, 0x2 vector)
    auto interleave = [&](auto V, auto K) {
        if constexpr (!F32) __builtin_amdgcn_sched_group_barrier(0x100, NP, 0);
#pragma unroll
        for (int k = 0; k < decltype(K)::value * NT; k++) {
            __builtin_amdgcn_sched_group_barrier(0x100, NP, 0);
#pragma unroll
            for (int m = 0; m < NM; m++) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, decltype(V)::value, 0);
            }
        }
    };
    auto step = [&](int t, int buf, float (&av)[4][8], const float (&an)[4][8], auto STEADY) {
        constexpr bool ST = decltype(STEADY)::value;
        const bool one = ST || t + kDwStep < t1, two = ST || t + 2 * kDwStep < t1;
        lds_barrier();
        const bool low = __builtin_amdgcn_readfirstlane(flag[buf]);   // the same for all waves
        if (low) fit_x(buf, std::false_type{});
        const float f_now = pow2(er);
        int en = er;
#pragma unroll
        for (int k = 0; k < 4; k++) {
#pragma unroll
            for (int j = 0; j < NT; j++) {
                f16x8 x[NP];
#pragma unroll
                for (int p = 0; p < NP; p++) x[p] = sx[buf][p][k][wn * NT + j][lane];
                // the smallest products first
                acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(s[1], x[0], acc[j], 0, 0, 0);
                if constexpr (NP > 1) acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(s[0], x[NP - 1], acc[j], 0, 0, 0);
                acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(s[0], x[0], acc[j], 0, 0, 0);
            }
            if (k < 3) {
                split_f16<2>(av[k < 3 ? k + 1 : 0], f_now, s);
            } else {   // the next step's, with the scale that fits it
                float m = row_max(an);
                m = fmaxf(m, __shfl_xor(m, 32, 64));
                en = m * f_now > kF16Max ? scale_exp(m, kDwTop) : er;
                split_f16<2>(an[0], pow2(en), s);
            }
            if (k == 0) {
                if (one) convert(buf ^ 1);
                if (two) load_x(t + 2 * kDwStep, STEADY);
                interleave(std::integral_constant<int, (F32 ? 128 : 112) / (NT * NM) + 1>{}, std::integral_constant<int, 1>{});
                __builtin_amdgcn_sched_barrier(0);   // x's loads no later
            }
        }
        if (two) load_a(t + 2 * kDwStep, av, STEADY);
        interleave(std::integral_constant<int, 120 / (3 * NT * NM) + 1>{}, std::integral_constant<int, 3>{});
        if (two) check_x(buf ^ 1);
        if (low)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const int d = shift[col_of(j)];
#pragma unroll
                for (int i = 0; i < 16; i++) acc[j][i] = __builtin_ldexpf(acc[j][i], d);
            }
        if (__any(en != er)) {
            const int d = en - er;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int di = __shfl(d, c_row(i, lane), 64);
#pragma unroll
                for (int j = 0; j < NT; j++) acc[j][i] = __builtin_ldexpf(acc[j][i], di);
            }
            er = en;
        }
    };
    load_x(t0, std::false_type{});
    load_a(t0, a[0], std::false_type{});
    fit_x(0, std::true_type{});
    convert(0);
    if (t0 + kDwStep < t1) {
        load_x(t0 + kDwStep, std::false_type{});
        load_a(t0 + kDwStep, a[1], std::false_type{});
        check_x(0);
    } else {
#pragma unroll
        for (int i = 0; i < 32; i++) a[1][i >> 3][i & 7] = 0.0f;
    }
    {
        const float m = row_max(a[0]);
        er = scale_exp(fmaxf(m, __shfl_xor(m, 32, 64)), kDwTop);
    }
    split_f16<2>(a[0][0], pow2(er), s);
    int t = t0;
#pragma unroll 1
    for (; t + 4 * kDwStep <= t1; t += 2 * kDwStep) {
        step(t, 0, a[0], a[1], std::true_type{});
        step(t + kDwStep, 1, a[1], a[0], std::true_type{});
    }
#pragma unroll 1
    for (; t < t1; t += 2 * kDwStep) {
        step(t, 0, a[0], a[1], std::false_type{});
        if (t + kDwStep < t1) step(t + kDwStep, 1, a[1], a[0], std::false_type{});
    }
    float *o = A.dw + (size_t)split * A.n_rows * kRgD;
    int ec[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) ec[j] = ecol[col_of(j)];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int row = r0 + c_row(i, lane), e = __shfl(er, c_row(i, lane), 64);
        float v[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) v[j] = __builtin_ldexpf(acc[j][i], -(e + ec[j]));
        if (row < A.n_expert) {
            if constexpr (NT > 1) {
#pragma unroll
                for (int j = 0; j < NT; j += 2)
                    *reinterpret_cast<float2 *>(o + (size_t)row * kRgD + n0 + col_of(j)) = make_float2(v[j], v[j + 1]);
            } else {
                o[(size_t)row * kRgD + n0 + col_of(0)] = v[0];
            }
        }
    }
    if (gate) {   // the waves hold the sums over their eighths of the tokens
        __syncthreads();
        scol[wave][2 * lane] = sg[0];
        scol[wave][2 * lane + 1] = sg[1];
        __syncthreads();
        const int col = 64 * wave + lane;
        if (col < kDwCols) {
            float v = scol[0][col];
#pragma unroll
            for (int k = 1; k < 8; k++) v += scol[k][col];
            o[(size_t)A.n_expert * kRgD + n0 + col] = v;
        }
    }
}

// ---- dx, up to 256 experts ----
// All of K fits in registers, so each token's gradients and each column of W are
// scaled by their own largest, to 2^14..2^15.  The same for a bf16 dx: one f16 per
// operand would be a third of the products, but 2^-10 of each term, which is above
// the result's own rounding where the terms cancel.
// Workgroup: 256 tokens, 32 per wave with their gradients in registers, against
// its part of the columns, 64 at a time through LDS.  4096 / 16384 fp32 tokens and
// 256 rows 24 / 64 us; the products alone, at the 1200 TFLOP/s that the chip holds
// on random operands, 11 / 43.
constexpr int kDxRows = 256, kDxCols = 64, kDxStages = kRgD / kDxCols;

template <int XF, int KS>   // K-steps of 16: 8 or 16
__global__ __launch_bounds__(512) void k_router_dx_split(ProductArgs A) {
    constexpr int NP = 2;                     // pieces of an operand
    constexpr int JW = KS / 8;                // K-steps of W that a wave converts
    constexpr int LDA = 68;                   // floats per staged row of 64: rows 4 banks apart
    __shared__ __align__(16) float sa[8][32 * LDA];
    __shared__ __align__(16) f16x8 sw[NP][2][KS][64];
    __shared__ __align__(16) float cmax[8][kDxCols];
    __shared__ __align__(16) int srow[8][32];
    __shared__ __align__(16) float sgate[8][32];
    const int lane = threadIdx.x & 63, half = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = xcd_order(blockIdx.x, gridDim.x);
    const int part = b % A.parts;
    const int tw = (int)(b / A.parts) * kDxRows + wave * 32;
    const int E = A.n_expert;
    const bool gate = A.n_rows > E;
    const int s0 = part * kDxStages / A.parts, s1 = (part + 1) * kDxStages / A.parts;

    // W through a buffer that ends with the last expert's row: rows past it
    // read as zeros
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(A.w), (short)0, E * kRgD * 4, 0x00020000);
    // dx through one that ends with the last token's row: rows past it are not
    // stored, without a branch around a store (which would make the next wait for
    // W one for every store as well)
    constexpr int XB = XF == Q36MOE_FMT_F32 ? 4 : 2;
    const __amdgpu_buffer_rsrc_t rdx = __builtin_amdgcn_make_buffer_rsrc(
        static_cast<uint8_t *>(A.dx) + (size_t)min(tw, A.T - 1) * kRgD * XB, (short)0, max(min(A.T - tw, 32), 0) * kRgD * XB, 0x00020000);
    float2 wr[JW][8];
    auto load_w = [&](int st) {
#pragma unroll
        for (int j = 0; j < JW; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(
                    rw, (16 * (wave * JW + j) + 8 * half + i) * (kRgD * 4) + 8 * c, st * kDxCols * 4, 0);
                wr[j][i] = make_float2(__uint_as_float(v[0]), __uint_as_float(v[1]));
            }
    };
    load_w(s0);

    // the wave's gradients to operand order, 64 columns at a time through its
    // own LDS; columns past the last expert are zeros
    f16x8 ga[KS][NP];
    {
        float4 g[2][8];   // two groups of 64 columns in flight
        auto load_g = [&](int p, float4 (&v4)[8]) {
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const float *row = A.dl + (size_t)min(tw + 4 * q + (lane >> 4), A.T - 1) * A.ld;
                const int k = 64 * p + 4 * (lane & 15);
                if (64 * p + 64 <= E) {
                    const f32x4 v = *reinterpret_cast<const f32x4_u *>(row + k);
                    v4[q] = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    const float v0 = row[min(k, E - 1)], v1 = row[min(k + 1, E - 1)], v2 = row[min(k + 2, E - 1)],
                                v3 = row[min(k + 3, E - 1)];
                    v4[q] = make_float4(k < E ? v0 : 0.0f, k + 1 < E ? v1 : 0.0f, k + 2 < E ? v2 : 0.0f, k + 3 < E ? v3 : 0.0f);
                }
            }
        };
        load_g(0, g[0]);
        load_g(1, g[1]);
        if (lane < 32) sgate[wave][lane] = gate ? A.dsh[(int64_t)min(tw + lane, A.T - 1) * A.ld_sh] : 0.0f;
        float raw[KS][8];
#pragma unroll
        for (int p = 0; p < KS / 4; p++) {
#pragma unroll
            for (int q = 0; q < 8; q++)
                *reinterpret_cast<float4 *>(&sa[wave][(4 * q + (lane >> 4)) * LDA + 4 * (lane & 15)]) = g[p & 1][q];
            if (p + 2 < KS / 4) load_g(p + 2, g[p & 1]);
            wave_sync();
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(&sa[wave][c * LDA + 16 * k + 8 * half + i]);
                    raw[4 * p + k][i] = v.x; raw[4 * p + k][i + 1] = v.y; raw[4 * p + k][i + 2] = v.z; raw[4 * p + k][i + 3] = v.w;
                }
            wave_sync();
        }
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(raw[k][i]));
        const int e = scale_exp(fmaxf(m, __shfl_xor(m, 32, 64)), 14);
        if (lane < 32) srow[wave][lane] = -e;
#pragma unroll
        for (int k = 0; k < KS; k++) split_f16<NP>(raw[k], pow2(e), ga[k]);
    }
    for (int st = s0; st < s1; st++) {
        const int n0 = st * kDxCols;
        float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
        for (int j = 0; j < JW; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                m0 = fmaxf(m0, fabsf(wr[j][i].x));
                m1 = fmaxf(m1, fabsf(wr[j][i].y));
            }
        m0 = fmaxf(m0, __shfl_xor(m0, 32, 64));
        m1 = fmaxf(m1, __shfl_xor(m1, 32, 64));
        if (lane < 32) *reinterpret_cast<float2 *>(&cmax[wave][2 * c]) = make_float2(m0, m1);
        lds_barrier();   // also: every wave has read the last stage's sw
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float2 v = *reinterpret_cast<const float2 *>(&cmax[k][2 * c]);
            m0 = fmaxf(m0, v.x);
            m1 = fmaxf(m1, v.y);
        }
        const int e0 = scale_exp(m0, 14), e1 = scale_exp(m1, 14);
#pragma unroll
        for (int j = 0; j < JW; j++) {
            float v[8];
            f16x8 h[NP];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = wr[j][i].x;
            split_f16<NP>(v, pow2(e0), h);
#pragma unroll
            for (int p = 0; p < NP; p++) sw[p][0][wave * JW + j][lane] = h[p];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = wr[j][i].y;
            split_f16<NP>(v, pow2(e1), h);
#pragma unroll
            for (int p = 0; p < NP; p++) sw[p][1][wave * JW + j][lane] = h[p];
        }
        if (st + 1 < s1) load_w(st + 1);
        float2 wg = make_float2(0.0f, 0.0f);
        if (gate) wg = *reinterpret_cast<const float2 *>(A.w + (size_t)E * kRgD + n0 + 2 * c);
        lds_barrier();
        f32x16 acc[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const f16x8 hi = sw[0][u][k][lane], lo = sw[1][u][k][lane];
                acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ga[k][1], hi, acc[u], 0, 0, 0);
                acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ga[k][0], lo, acc[u], 0, 0, 0);
                acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ga[k][0], hi, acc[u], 0, 0, 0);
            }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int r = c_row(i, lane);
            const int er = srow[wave][r];
            const float g = sgate[wave][r];
            const float v0 = fmaf(g, wg.x, __builtin_ldexpf(acc[0][i], er - e0)), v1 = fmaf(g, wg.y, __builtin_ldexpf(acc[1][i], er - e1));
            if constexpr (XF == Q36MOE_FMT_F32)
                __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(v0), __float_as_uint(v1)}, rdx, r * kRgD * 4 + 8 * c, n0 * 4, 0);
            else
                __builtin_amdgcn_raw_buffer_store_b32(bf16_pair(v0, v1), rdx, r * kRgD * 2 + 4 * c, n0 * 2, 0);
        }
    }
}

constexpr int kCUs = 256;

// Tokens from which the split operands pay.  Their time is nearly flat there (two
// launches of one workgroup per CU, and the sum of dW's splits), that of the fp32
// tiles grows with the tokens.  us of both gradients, fp32 x (fp32 tiles / split):
// 256 + 1 rows, 512 tokens 27 / 30, 700 35 / 32, 1024 46 / 33; 128 rows, 700
// 19 / 22, 1024 24 / 25, 1400 31 / 28; 60 rows, 1024 20 / 25, 1400 27 / 27, 2048 36 / 29.
int split_from(int n_expert) { return n_expert > 128 ? 640 : n_expert > 64 ? 1024 : 1400; }

// Waves along the router rows in k_router_dw_split.
int dw_mw(int n_expert) { return n_expert <= 64 ? 2 : n_expert <= 128 ? 4 : 8; }

// Splits of the tokens: one workgroup per CU, and at least two steps each.
int dw_span(int T, int n_expert) {
    const int mw = dw_mw(n_expert);
    const int tiles = kRgD / kDwCols * ((n_expert + 32 * mw - 1) / (32 * mw));
    const int want = kCUs / tiles > 1 ? kCUs / tiles : 1;
    const int span = ((T + want - 1) / want + kDwStep - 1) / kDwStep * kDwStep;
    return span > 2 * kDwStep ? span : 2 * kDwStep;
}
int dw_splits(int T, int n_expert) {
    if (T < split_from(n_expert)) return 1;
    const int span = dw_span(T, n_expert);
    return (T + span - 1) / span;
}

template <int XF>
void launch_product(const ProductArgs &P, float *dw, float *ws, hipStream_t s) {
    ProductArgs A = P;
    const bool many = A.T >= split_from(A.n_expert);
    const bool dw_many = dw && many, dx_many = A.dx && many && A.n_expert <= 256;
    if (dw_many) {
        const int mw = dw_mw(A.n_expert), splits = dw_splits(A.T, A.n_expert);
        A.span = dw_span(A.T, A.n_expert);
        A.dw = splits == 1 ? dw : ws;
        const dim3 g((unsigned)(splits * (kRgD / kDwCols) * ((A.n_expert + 32 * mw - 1) / (32 * mw))));
        if (mw == 2) hipLaunchKernelGGL((k_router_dw_split<XF, 2>), g, dim3(512), 0, s, A);
        else if (mw == 4) hipLaunchKernelGGL((k_router_dw_split<XF, 4>), g, dim3(512), 0, s, A);
        else hipLaunchKernelGGL((k_router_dw_split<XF, 8>), g, dim3(512), 0, s, A);
        if (splits > 1) sum_partials(ws, splits, (size_t)A.n_rows * kRgD, (size_t)A.n_rows * kRgD, dw, nullptr, s);
    }
    if (dx_many) {
        const int blocks = (A.T + kDxRows - 1) / kDxRows;
        A.parts = blocks >= kCUs ? 1 : kCUs / blocks < kDxStages ? kCUs / blocks : kDxStages;
        const dim3 g((unsigned)(blocks * A.parts));
        if (A.n_expert <= 128) hipLaunchKernelGGL((k_router_dx_split<XF, 8>), g, dim3(512), 0, s, A);
        else hipLaunchKernelGGL((k_router_dx_split<XF, 16>), g, dim3(512), 0, s, A);
    }
    const int nw = dw && !dw_many ? (A.n_rows + 31) / 32 * (kRgD / kF32Cols) : 0;
    const int nx = A.dx && !dx_many ? (A.T + 31) / 32 * (kRgD / kF32Cols) : 0;
    if (nw + nx) {
        A.dw = dw;
        A.nw = nw;
        hipLaunchKernelGGL(k_router_grad_f32<XF>, dim3((unsigned)(nw + nx)), dim3(256), 0, s, A);
    }
}

}  // namespace

extern "C" {

size_t q36moe_balance_loss_workspace(int T, int n_expert) {
    if (T < 1 || n_expert < 1 || n_expert > kMaxE) return 0;
    const int nb = balance_groups(T);
    return nb == 1 ? 0 : balance_part_bytes(nb, n_expert) + sizeof(BalanceJoin);
}

int q36moe_balance_loss(const float *logits, int ld, const int32_t *idx, const uint8_t *mask, int T, int n_expert, int k,
                        float coef, int32_t *counts, float *psum, float *loss, void *ws, size_t ws_bytes, void *stream) {
    if (T < 0 || n_expert < 1 || n_expert > kMaxE || ld < n_expert || k < 1 || k > kMaxK || k > n_expert)
        return Q36MOE_EINVAL;
    if (!counts || !psum || !loss || (T > 0 && (!logits || !idx))) return Q36MOE_EINVAL;
    if ((int64_t)T * k > INT32_MAX) return Q36MOE_EINVAL;   // counts are 32 bits
    const size_t need = q36moe_balance_loss_workspace(T, n_expert);
    if (!workspace_ok(ws, ws_bytes, need)) return Q36MOE_EINVAL;
    BalanceArgs A{logits, idx, mask, ld, T, n_expert, k, 0, coef, counts, psum, loss, static_cast<float2 *>(ws)};
    const int nb = T ? balance_groups(T) : 1;
    A.chunk = (int)(((int64_t)T + nb - 1) / nb);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n_expert <= 64) hipLaunchKernelGGL(k_balance<1>, dim3(nb), dim3(64 * kBalW), 0, s, A);
    else hipLaunchKernelGGL(k_balance<4>, dim3(nb), dim3(64 * kBalW), 0, s, A);
    if (nb > 1) hipLaunchKernelGGL(k_balance_join, dim3((n_expert + kJoinE) / kJoinE), dim3(256), 0, s, A, nb);
    return hip_status(hipGetLastError());
}

int q36moe_router_topk_backward(const float *logits, int ld, const int32_t *idx, const float *dwt, const int32_t *counts,
                                const uint8_t *mask, const float *dloss, int T, int n_expert, int k, float scale, int renorm,
                                float coef, float *dlogits, int ld_d, void *stream) {
    if (T < 0 || n_expert < 1 || n_expert > kMaxE || ld < n_expert || ld_d < n_expert || k < 1 || k > kMaxK || k > n_expert ||
        (!dwt && !counts))
        return Q36MOE_EINVAL;
    if (T == 0) return Q36MOE_OK;
    if (!logits || !dlogits || (dwt && !idx)) return Q36MOE_EINVAL;
    const LogitGradArgs A{logits, idx, dwt, counts, mask, dloss, dlogits, ld, ld_d, T, n_expert, k, renorm, scale, coef};
    const int64_t nb = ((int64_t)T + 15) / 16;
    const dim3 g((unsigned)(nb < 4096 ? nb : 4096));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool full = counts || !renorm;
    if (n_expert <= 64) {
        if (full) hipLaunchKernelGGL((k_logit_grad<1, true>), g, dim3(256), 0, s, A);
        else hipLaunchKernelGGL((k_logit_grad<1, false>), g, dim3(256), 0, s, A);
    } else {
        if (full) hipLaunchKernelGGL((k_logit_grad<4, true>), g, dim3(256), 0, s, A);
        else hipLaunchKernelGGL((k_logit_grad<4, false>), g, dim3(256), 0, s, A);
    }
    return hip_status(hipGetLastError());
}

size_t q36moe_router_logits_backward_workspace(int T, int n_rows) {
    if (T < 1 || n_rows < 1 || T > kMaxRouterT) return 0;
    const int a = dw_splits(T, n_rows), b = n_rows > 1 ? dw_splits(T, n_rows - 1) : 1, n = a > b ? a : b;   // without and with a shared gate
    return n == 1 ? 0 : (size_t)n * n_rows * kRgD * sizeof(float);
}

int q36moe_router_logits_backward(const float *w, int n_rows, int n_expert, const void *x, int x_fmt, int T, int d_model,
                                  const float *dlogits, int ld, const float *dshg, int ld_shg, float *dw, void *dx, void *ws,
                                  size_t ws_bytes, void *stream) {
    if (T < 0 || T > kMaxRouterT || d_model != kRgD || n_expert < 1 || n_rows < n_expert || n_rows > n_expert + 1 ||
        n_rows > kMaxRouterRows || ld < n_expert || ld > kMaxRouterLd || (x_fmt != Q36MOE_FMT_F32 && x_fmt != Q36MOE_FMT_BF16) || (!dw && !dx) ||
        ld_shg < 0)
        return Q36MOE_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (T == 0) {   // sums of nothing
        if (!dw) return Q36MOE_OK;
        sum_partials(nullptr, 0, (size_t)n_rows * kRgD, (size_t)n_rows * kRgD, dw, nullptr, s);
        return hip_status(hipGetLastError());
    }
    if (!dlogits || (dw && !x) || (dx && !w) || (n_rows > n_expert && !dshg)) return Q36MOE_EINVAL;
    const size_t need = dw ? q36moe_router_logits_backward_workspace(T, n_rows) : 0;
    if (!workspace_ok(ws, ws_bytes, need)) return Q36MOE_EINVAL;
    if (((uintptr_t)x | (uintptr_t)dx) & 3) return Q36MOE_EINVAL;   // pairs of bf16
    ProductArgs A{};
    A.w = w; A.dl = dlogits; A.dsh = dshg; A.x = x; A.dx = dx;
    A.ld = ld; A.ld_sh = ld_shg ? ld_shg : 1;
    A.n_rows = n_rows; A.n_expert = n_expert; A.T = T;
    if (x_fmt == Q36MOE_FMT_F32) launch_product<Q36MOE_FMT_F32>(A, dw, static_cast<float *>(ws), s);
    else launch_product<Q36MOE_FMT_BF16>(A, dw, static_cast<float *>(ws), s);
    return hip_status(hipGetLastError());
}

}  // extern "C"
