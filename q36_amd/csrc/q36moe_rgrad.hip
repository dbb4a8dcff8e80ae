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

namespace {

constexpr int kMaxE = 256, kMaxK = 8;

// exp(x) for x <= 0 as 2^hi * (1 + lo ln 2), hi + lo = x log2(e) to 48 bits:
// about 1 ulp however large -x is.
__device__ __forceinline__ float exp_neg(float x) {
    constexpr float kL = 1.44269502162933349609f, kLl = 1.92596299112661746887e-8f;   // log2(e) in two floats
    const float hi = x * kL;
    const float lo = fmaf(x, kLl, fmaf(x, kL, -hi));
    const float e = __builtin_amdgcn_exp2f(hi);
    // x = -inf gives lo = NaN where e is 0 already
    return e == 0.0f ? 0.0f : fmaf(e, lo * 0.693147180559945309417f, e);
}

// Softmax of a token's logits by 16 lanes; lane l holds experts l + 16 i, -inf
// past the last one.  A row of -inf has no probabilities: all 0.
template <int NI>
__device__ __forceinline__ void softmax16(float (&v)[NI]) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < NI; i++) m = fmaxf(m, v[i]);
    m = max16(m);
    m = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; i++) {
        v[i] = exp_neg(v[i] - m);
        s += v[i];
    }
    s = sum16(s);
    const float inv = s == 0.0f ? 0.0f : 1.0f / s;   // a NaN stays one
#pragma unroll
    for (int i = 0; i < NI; i++) v[i] *= inv;
}

template <int NI>
__device__ __forceinline__ void load_logits(const float *__restrict__ row, int E, int l, float (&v)[NI]) {
#pragma unroll
    for (int i = 0; i < NI; i++) v[i] = row[min(l + 16 * i, E - 1)];
#pragma unroll
    for (int i = 0; i < NI; i++) v[i] = l + 16 * i < E ? v[i] : -INFINITY;
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
    float *part;               // [workgroups][E] sums, then [workgroups][E + 1] counts
};

// loss from counts and sums by one workgroup, in 64 bits: counts times sums of
// probabilities over many tokens.
__device__ __forceinline__ void balance_of(const BalanceArgs &A, const int32_t *cnt, const float *ps, double *red) {
    if (threadIdx.x < 64) {
        double s = 0.0;
        for (int e = threadIdx.x; e < A.E; e += 64) s += (double)cnt[e] * (double)ps[e];
        red[threadIdx.x] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int i = 0; i < 64; i++) s += red[i];
        const double n = (double)cnt[A.E];
        *A.loss = n > 0.0 ? (float)((double)A.coef * A.E * s / ((double)A.k * n * n)) : 0.0f;
    }
}

constexpr int kBalW = 16;   // waves per workgroup

// 16 lanes per token, 64 tokens of the workgroup's run at a time.
template <int NI>
__global__ __launch_bounds__(64 * kBalW) void k_balance(BalanceArgs A) {
    __shared__ float ps[kBalW][16 * NI];
    __shared__ int32_t cnt[kMaxE + 1];
    __shared__ double red[64];
    const int tid = threadIdx.x, l = tid & 15, wave = tid >> 6;
    const int64_t t0 = (int64_t)blockIdx.x * A.chunk, t1 = min(t0 + A.chunk, (int64_t)A.T);
    for (int e = tid; e <= A.E; e += 64 * kBalW) cnt[e] = 0;
    float acc[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) acc[i] = 0.0f;
    for (int64_t t = t0 + (tid >> 4); t < t1; t += 4 * kBalW) {
        if (A.mask && !A.mask[t]) continue;
        float v[NI];
        load_logits(A.logits + (size_t)t * A.ld, A.E, l, v);
        softmax16(v);
#pragma unroll
        for (int i = 0; i < NI; i++) acc[i] += v[i];
    }
    __syncthreads();   // cnt cleared
    int live = 0;
    for (int64_t t = t0 + tid; t < t1; t += 64 * kBalW) {
        if (A.mask && !A.mask[t]) continue;
        live++;
        for (int s = 0; s < A.k; s++) {
            const int e = A.idx[(size_t)t * A.k + s];
            if ((unsigned)e < (unsigned)A.E) atomicAdd(&cnt[e], 1);
        }
    }
    if (live) atomicAdd(&cnt[A.E], live);
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const float s = sum_rows4(acc[i]);
        if ((tid & 63) < 16) ps[wave][l + 16 * i] = s;
    }
    __syncthreads();
    const bool all = gridDim.x == 1;
    float *po = all ? A.psum : A.part + (size_t)blockIdx.x * A.E;
    int32_t *co = all ? A.counts
                      : reinterpret_cast<int32_t *>(A.part + (size_t)gridDim.x * A.E) + (size_t)blockIdx.x * (A.E + 1);
    for (int e = tid; e < A.E; e += 64 * kBalW) {
        float s = ps[0][e];
#pragma unroll
        for (int w = 1; w < kBalW; w++) s += ps[w][e];
        po[e] = s;
        ps[0][e] = s;
    }
    for (int e = tid; e <= A.E; e += 64 * kBalW) co[e] = cnt[e];
    if (all) {
        __syncthreads();
        balance_of(A, cnt, ps[0], red);
    }
}

// The workgroups' parts to counts, sums and loss: thread (group of parts, expert).
__global__ __launch_bounds__(1024) void k_balance_join(BalanceArgs A, int nb) {
    __shared__ float ps[4][kMaxE];
    __shared__ int32_t cs[4][kMaxE + 1];
    __shared__ double red[64];
    const int e = threadIdx.x & 255, g = threadIdx.x >> 8;
    const int32_t *cpart = reinterpret_cast<const int32_t *>(A.part + (size_t)nb * A.E);
    if (e < A.E) {
        float s = 0.0f;
        int32_t c = 0;
#pragma unroll 8
        for (int b = g; b < nb; b += 4) {
            s += A.part[(size_t)b * A.E + e];
            c += cpart[(size_t)b * (A.E + 1) + e];
        }
        ps[g][e] = s;
        cs[g][e] = c;
    }
    if (e == 0) {
        int32_t c = 0;
        for (int b = g; b < nb; b += 4) c += cpart[(size_t)b * (A.E + 1) + A.E];
        cs[g][A.E] = c;
    }
    __syncthreads();
    for (int i = threadIdx.x; i <= A.E; i += 1024) {
        const int32_t c = cs[0][i] + cs[1][i] + cs[2][i] + cs[3][i];
        cs[0][i] = c;
        A.counts[i] = c;
        if (i < A.E) {
            const float s = (ps[0][i] + ps[1][i]) + (ps[2][i] + ps[3][i]);
            ps[0][i] = s;
            A.psum[i] = s;
        }
    }
    __syncthreads();
    balance_of(A, cs[0], ps[0], red);
}

// Workgroups: one up to 256 tokens (no second launch), then 128 tokens each up
// to 128 of them, whose parts one workgroup still joins in a few microseconds.
int balance_groups(int T) {
    if (T <= 256) return 1;
    const int n = (int)(((int64_t)T + 127) / 128);
    return n < 128 ? n : 128;
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

// 16 lanes per token.  The softmax over all experts is formed only where the
// balance loss or weights that are not renormalised ask for it; the gradients
// of the picks are added to their experts by the lanes that hold them, in slot
// order, so an expert that was picked twice gets both.
template <int NI>
__global__ __launch_bounds__(256) void k_logit_grad(LogitGradArgs A) {
    const int l = threadIdx.x & 15;
    float f[NI];
    float gain = 0.0f;
    if (A.counts) {
        const float n = (float)A.counts[A.E];
        const float den = n * (float)A.k;
        gain = n > 0.0f ? A.coef * (float)A.E / n * (A.dloss ? *A.dloss : 1.0f) : 0.0f;
#pragma unroll
        for (int i = 0; i < NI; i++) f[i] = l + 16 * i < A.E && n > 0.0f ? (float)A.counts[l + 16 * i] / den : 0.0f;
    }
    const bool full = A.counts || (A.dwt && !A.renorm);
    for (int64_t t = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); t < A.T; t += (int64_t)gridDim.x * 16) {
        float o[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) o[i] = 0.0f;
        if (!A.mask || A.mask[t]) {
            const float *row = A.logits + (size_t)t * A.ld;
            float p[NI];
            if (full) {
                load_logits(row, A.E, l, p);
                softmax16(p);
            }
            if (A.counts) {
                float d = 0.0f;
#pragma unroll
                for (int i = 0; i < NI; i++) d = fmaf(p[i], f[i], d);
                d = sum16(d);
#pragma unroll
                for (int i = 0; i < NI; i++) o[i] = gain * p[i] * (f[i] - d);
            }
            if (A.dwt) {
                // lane s < k holds slot s; a slot whose index names no expert is none
                int e = -1;
                float up = 0.0f;
                if (l < A.k) {
                    e = A.idx[(size_t)t * A.k + l];
                    e = (unsigned)e < (unsigned)A.E ? e : -1;
                    up = e >= 0 ? A.dwt[(size_t)t * A.k + l] * A.scale : 0.0f;
                }
                float s = up;
                if (A.renorm) {
                    float q[1] = {e >= 0 ? row[e] : -INFINITY};
                    softmax16(q);
                    s = q[0] * (up - sum16(q[0] * up));
                    s = e >= 0 ? s : 0.0f;
                }
                float u[NI];
#pragma unroll
                for (int i = 0; i < NI; i++) u[i] = 0.0f;
#pragma unroll
                for (int j = 0; j < kMaxK; j++) {
                    if (j < A.k) {
                        const int ej = __shfl(e, j, 16);
                        const float sj = __shfl(s, j, 16);
#pragma unroll
                        for (int i = 0; i < NI; i++) u[i] += ej == l + 16 * i ? sj : 0.0f;
                    }
                }
                if (A.renorm) {
#pragma unroll
                    for (int i = 0; i < NI; i++) o[i] += u[i];
                } else {
                    float d = 0.0f;
#pragma unroll
                    for (int i = 0; i < NI; i++) d = fmaf(p[i], u[i], d);
                    d = sum16(d);
#pragma unroll
                    for (int i = 0; i < NI; i++) o[i] = fmaf(p[i], u[i] - d, o[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NI; i++)
            if (l + 16 * i < A.E) A.out[(size_t)t * A.ldo + l + 16 * i] = o[i];
    }
}

// ---------------------------------------------------------------------------
// gradients of the router product
// ---------------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kRgD = 2048;
constexpr int kMaxRouterT = 1 << 25, kMaxRouterRows = 1 << 20;

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

// Workgroup barrier for LDS data only: prefetched global loads stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Workgroup b of n in an order in which those of one XCD (b % 8) are neighbours.
__device__ __forceinline__ int xcd_order(int b, int n) { return (n & 7) ? b : (b & 7) * (n >> 3) + (b >> 3); }

// ---- few tokens: fp32 MFMA ----
// v_mfma_f32_32x32x2_f32: lane L holds row (A) or column (B) L % 32 at K element
// L / 32.  One 32 x 32 tile per wave, no LDS: the products cost 64 cycles each,
// and a wave's operands come straight from the caches, the next batch of loads
// issued before the products of this one.  dW and dx share the launch.
constexpr int kF32Batch = 16;

template <int XF>
__device__ __forceinline__ float load_x(const void *x, size_t at) {
    if constexpr (XF == Q36MOE_FMT_F32) return static_cast<const float *>(x)[at];
    else return __uint_as_float((uint32_t)static_cast<const uint16_t *>(x)[at] << 16);
}

template <int XF>
__device__ __forceinline__ void f32_dw_tile(const ProductArgs &A, int rt, int d0) {
    constexpr int U = kF32Batch;
    const int lane = threadIdx.x & 63, half = lane >> 5, c = lane & 31;
    const int r = min(rt * 32 + c, A.n_rows - 1);
    const bool sh = r >= A.n_expert;
    const float *col = sh ? A.dsh : A.dl + r;
    const int64_t step = sh ? A.ld_sh : A.ld;
    f32x16 acc = {};
    float a[2][U], b[2][U];
    auto load = [&](int t, float (&av)[U], float (&bv)[U]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int tc = min(t + 2 * u + half, A.T - 1);
            av[u] = col[tc * step];
            bv[u] = load_x<XF>(A.x, (size_t)tc * kRgD + d0 + c);
        }
    };
    auto products = [&](int t, const float (&av)[U], const float (&bv)[U]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool in = t + 2 * u + half < A.T;   // past the end the last token again, as zeros
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? av[u] : 0.0f, in ? bv[u] : 0.0f, acc, 0, 0, 0);
        }
    };
    load(0, a[0], b[0]);
    for (int t = 0; t < A.T; t += 4 * U) {
        if (t + 2 * U < A.T) load(t + 2 * U, a[1], b[1]);
        products(t, a[0], b[0]);
        if (t + 2 * U < A.T) {
            if (t + 4 * U < A.T) load(t + 4 * U, a[0], b[0]);
            products(t + 2 * U, a[1], b[1]);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int row = rt * 32 + c_row(i, lane);
        if (row < A.n_rows) A.dw[(size_t)row * kRgD + d0 + c] = acc[i];
    }
}

// Lane half h of a step of 8 rows holds rows 4h..4h+3 of both operands.
template <int XF>
__device__ __forceinline__ void f32_dx_tile(const ProductArgs &A, int tb, int d0) {
    constexpr int U = kF32Batch / 4;
    const int lane = threadIdx.x & 63, half = lane >> 5, c = lane & 31;
    const int t = min(tb + c, A.T - 1);
    const float *row = A.dl + (size_t)t * A.ld, *col = A.w + d0 + c;
    f32x16 acc = {};
    float a[2][U][4], b[2][U][4];
    auto load = [&](int r0, float (&av)[U][4], float (&bv)[U][4]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = r0 + 8 * u + 4 * half;
            load_row<Q36MOE_FMT_F32>(row, r, av[u]);
#pragma unroll
            for (int i = 0; i < 4; i++) bv[u][i] = col[(size_t)(r + i) * kRgD];
        }
    };
    auto products = [&](const float (&av)[U][4], const float (&bv)[U][4]) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(av[u][i], bv[u][i], acc, 0, 0, 0);
    };
    const int whole = A.n_expert & ~(8 * U - 1);
    if (whole) load(0, a[0], b[0]);
    for (int r0 = 0; r0 < whole; r0 += 16 * U) {
        if (r0 + 8 * U < whole) load(r0 + 8 * U, a[1], b[1]);
        products(a[0], b[0]);
        if (r0 + 8 * U < whole) {
            if (r0 + 16 * U < whole) load(r0 + 16 * U, a[0], b[0]);
            products(a[1], b[1]);
        }
    }
    // the rows left over, the shared gate's among them
    for (int r0 = whole; r0 < A.n_rows; r0 += 16) {
        float av[8], bv[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int r = min(r0 + 2 * u + half, A.n_rows - 1);
            av[u] = r < A.n_expert ? row[r] : A.dsh[(size_t)t * A.ld_sh];
            bv[u] = col[(size_t)r * kRgD];
        }
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const bool in = r0 + 2 * u + half < A.n_rows;
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? av[u] : 0.0f, in ? bv[u] : 0.0f, acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int tt = tb + c_row(i, lane);
        if (tt < A.T) store_one<XF>(A.dx, (size_t)tt * kRgD + d0 + c, acc[i]);
    }
}

constexpr int kF32Cols = 128;   // columns per workgroup, 32 per wave

template <int XF>
__global__ __launch_bounds__(256) void k_router_grad_f32(ProductArgs A) {
    const int wave = threadIdx.x >> 6;
    const bool is_dw = (int)blockIdx.x < A.nw;
    const int b = is_dw ? blockIdx.x : blockIdx.x - A.nw;
    const int d0 = b % (kRgD / kF32Cols) * kF32Cols + wave * 32, tile = b / (kRgD / kF32Cols);
    if (is_dw) f32_dw_tile<XF>(A, tile, d0);
    else f32_dx_tile<XF>(A, tile * 32, d0);
}

// ---- dW of many tokens: operands split into bf16 ----
// v_mfma_f32_32x32x16_bf16 takes 32 cycles for eight times the products of the
// fp32 MFMA.  An fp32 value is the sum of three bf16 (8 bits each, the rests
// exact); of the nine products of two such sums the six down to 2^-16 of the
// largest are formed, what is left out is 2^-24 of each product.  A bf16 x is
// one piece, which leaves three products.  No scaling: bf16 has fp32's range.
struct Pieces { bf16x8 p[3]; };

__device__ __forceinline__ Pieces split3(const float (&v)[8]) {
    Pieces s;
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = v[i];
#pragma unroll
    for (int k = 0; k < 3; k++) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const bf16x2 h = __builtin_convertvector((f32x2{r[i], r[i + 1]}), bf16x2);
            s.p[k][i] = h[0];
            s.p[k][i + 1] = h[1];
            const uint32_t u = __builtin_bit_cast(uint32_t, h);
            r[i] -= bf16_lo(u);
            r[i + 1] -= bf16_hi(u);
        }
    }
    return s;
}

// Workgroup: 32 MW router rows x 128 columns over the tokens of its split, 8
// waves as MW x 8 / MW.  Lane L of an operand holds row (column) L % 32 at K
// elements (tokens) 8 (L / 32)..+7.  A wave reads its rows of the logits'
// gradient straight into that order (32 neighbouring values per load) and splits
// them itself; x is split once per workgroup and shared through LDS in operand
// order, two buffers, one barrier per 64 tokens.  The columns of MFMA tiles 2q
// and 2q + 1 interleave, so pairs of columns load and store as 8 bytes.
// The shared gate's row is an fp32 sum beside the conversion of x.
constexpr int kDwCols = 128, kDwStep = 64;

template <int XF, int MW>
__global__ __launch_bounds__(512) void k_router_dw_split(ProductArgs A) {
    constexpr bool F32 = XF == Q36MOE_FMT_F32;
    constexpr int NP = F32 ? 3 : 1;           // pieces of x
    constexpr int NT = MW / 2;                // tiles per wave
    __shared__ __align__(16) bf16x8 sx[2][NP][4][4][64];
    __shared__ float ssh[8][kDwCols];
    const int lane = threadIdx.x & 63, half = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % MW, wn = wave / MW;
    const int mblocks = (A.n_expert + 32 * MW - 1) / (32 * MW), tiles = kRgD / kDwCols * mblocks;
    const int b = xcd_order(blockIdx.x, gridDim.x);
    const int split = b / tiles, n0 = b % tiles % (kRgD / kDwCols) * kDwCols, mb = b % tiles / (kRgD / kDwCols);
    const int r0 = (mb * MW + wm) * 32;
    const int t0 = split * A.span, t1 = min(t0 + A.span, A.T);
    const bool gate = A.n_rows > A.n_expert && mb == 0;
    const float *dl = A.dl + min(r0 + c, A.n_expert - 1);

    f32x16 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j] = f32x16{};
    float sg[2] = {0.0f, 0.0f};
    float a[2][4][8];
    uint32_t xr[8][F32 ? 2 : 1];              // tokens t + 8 wave + i, columns n0 + 2 lane, + 1
    float sh[8];

    auto load = [&](int t, float (&av)[4][8]) {
        const int tx = t + 8 * wave;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const size_t o = (size_t)min(tx + i, A.T - 1) * kRgD + n0 + 2 * lane;
            if constexpr (F32) {
                const float2 v = *reinterpret_cast<const float2 *>(static_cast<const float *>(A.x) + o);
                xr[i][0] = __float_as_uint(v.x);
                xr[i][1] = __float_as_uint(v.y);
            } else {
                xr[i][0] = *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(A.x) + o);
            }
        }
        if (gate)
#pragma unroll
            for (int i = 0; i < 8; i++) sh[i] = A.dsh[(int64_t)min(tx + i, A.T - 1) * A.ld_sh];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) av[k][i] = dl[(int64_t)min(t + 16 * k + 8 * half + i, A.T - 1) * A.ld];
    };
    // this step's x to LDS; tokens past the split's end count as zeros
    auto convert = [&](int t, int buf) {
        const int left = t1 - (t + 8 * wave);
        if (left < 8)
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int u = 0; u < (F32 ? 2 : 1); u++) xr[i][u] = i < left ? xr[i][u] : 0u;
        const int k = wave >> 1, at = (lane & 31) + 32 * (wave & 1), q = lane >> 5;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            if constexpr (F32) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = __uint_as_float(xr[i][u]);
                const Pieces s = split3(v);
#pragma unroll
                for (int p = 0; p < NP; p++) sx[buf][p][k][2 * q + u][at] = s.p[p];
                if (gate)
#pragma unroll
                    for (int i = 0; i < 8; i++) sg[u] = fmaf(i < left ? sh[i] : 0.0f, v[i], sg[u]);
            } else {
                u32x4_u h;
#pragma unroll
                for (int i = 0; i < 4; i++)   // the columns' halves of two tokens side by side
                    h[i] = __builtin_amdgcn_perm(xr[2 * i + 1][0], xr[2 * i][0], u ? 0x07060302u : 0x05040100u);
                sx[buf][0][k][2 * q + u][at] = __builtin_bit_cast(bf16x8, h);
                if (gate)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        sg[u] = fmaf(i < left ? sh[i] : 0.0f, u ? bf16_hi(xr[i][0]) : bf16_lo(xr[i][0]), sg[u]);
            }
        }
    };
    auto products = [&](int t, int buf, float (&av)[4][8]) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (t + 64 > t1)
#pragma unroll
                for (int i = 0; i < 8; i++) av[k][i] = t + 16 * k + 8 * half + i < t1 ? av[k][i] : 0.0f;
            const Pieces s = split3(av[k]);
#pragma unroll
            for (int j = 0; j < NT; j++) {
                bf16x8 x[NP];
#pragma unroll
                for (int p = 0; p < NP; p++) x[p] = sx[buf][p][k][wn * NT + j][lane];
                // the smallest products first
#pragma unroll
                for (int o = 2; o >= 0; o--)
#pragma unroll
                    for (int p = 0; p <= o; p++)
                        if (p < NP) acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(s.p[o - p], x[p], acc[j], 0, 0, 0);
            }
        }
    };
    load(t0, a[0]);
    for (int t = t0; t < t1; t += 2 * kDwStep) {
        convert(t, 0);
        if (t + kDwStep < t1) load(t + kDwStep, a[1]);
        lds_barrier();
        products(t, 0, a[0]);
        if (t + kDwStep < t1) {
            convert(t + kDwStep, 1);
            if (t + 2 * kDwStep < t1) load(t + 2 * kDwStep, a[0]);
            lds_barrier();
            products(t + kDwStep, 1, a[1]);
        }
    }
    float *o = A.dw + (size_t)split * A.n_rows * kRgD;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int row = r0 + c_row(i, lane);
        if (row < A.n_expert) {
            if constexpr (NT > 1) {
#pragma unroll
                for (int j = 0; j < NT; j += 2)
                    *reinterpret_cast<float2 *>(o + (size_t)row * kRgD + n0 + 32 * (wn * NT + j) + 2 * c) =
                        make_float2(acc[j][i], acc[j + 1][i]);
            } else {
                o[(size_t)row * kRgD + n0 + 64 * (wn >> 1) + 2 * c + (wn & 1)] = acc[0][i];
            }
        }
    }
    if (gate) {   // the waves hold the sums over their eighths of the tokens
        ssh[wave][2 * lane] = sg[0];
        ssh[wave][2 * lane + 1] = sg[1];
        __syncthreads();
        if (threadIdx.x < kDwCols) {
            float v = ssh[0][threadIdx.x];
#pragma unroll
            for (int k = 1; k < 8; k++) v += ssh[k][threadIdx.x];
            o[(size_t)A.n_expert * kRgD + n0 + threadIdx.x] = v;
        }
    }
}

// ---- dx of many tokens, up to 256 experts: operands split into f16 ----
// All of K fits in registers, so each token's gradients and each column of W
// can be scaled by a power of two that puts the largest at 2^14..2^15: two f16
// (11 bits each) then hold a value to 2^-22 of itself, or to 2^-40 of the
// largest where that is more, and three products of v_mfma_f32_32x32x16_f16
// give fp32's exactness (the fourth is 2^-22 of the first).
// Workgroup: 256 tokens, 32 per wave with their gradients in registers, against
// its part of the columns, 64 at a time through LDS.
__device__ __forceinline__ int scale_exp(float amax) {   // amax * 2^this is in [2^14, 2^15)
    const int e = (int)(__float_as_uint(amax) >> 23);     // 0 for zero and denormals, 255 for inf
    return 141 - max(e, 1);
}

__device__ __forceinline__ void split_f16(const float (&v)[8], int e, f16x8 (&p)[2]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float s = __builtin_ldexpf(v[i], e);
        p[0][i] = (_Float16)s;
        p[1][i] = (_Float16)(s - (float)p[0][i]);
    }
}

constexpr int kDxRows = 256, kDxCols = 64, kDxStages = kRgD / kDxCols;

template <int XF, int KS>   // K-steps of 16: 8 or 16
__global__ __launch_bounds__(512) void k_router_dx_split(ProductArgs A) {
    constexpr int JW = KS / 8;                // K-steps of W that a wave converts
    constexpr int LDA = 68;                   // floats per staged row of 64: rows 4 banks apart
    __shared__ __align__(16) float sa[8][32 * LDA];
    __shared__ __align__(16) f16x8 sw[2][2][KS][64];
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
    f16x8 ga[KS][2];
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
        const int e = scale_exp(fmaxf(m, __shfl_xor(m, 32, 64)));
        if (lane < 32) srow[wave][lane] = -e;
#pragma unroll
        for (int k = 0; k < KS; k++) split_f16(raw[k], e, ga[k]);
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
        const int e0 = scale_exp(m0), e1 = scale_exp(m1);
#pragma unroll
        for (int j = 0; j < JW; j++) {
            float v[8];
            f16x8 h[2];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = wr[j][i].x;
            split_f16(v, e0, h);
#pragma unroll
            for (int p = 0; p < 2; p++) sw[p][0][wave * JW + j][lane] = h[p];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = wr[j][i].y;
            split_f16(v, e1, h);
#pragma unroll
            for (int p = 0; p < 2; p++) sw[p][1][wave * JW + j][lane] = h[p];
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
            const int r = c_row(i, lane), t = tw + r;
            const int er = srow[wave][r];
            const float g = sgate[wave][r];
            const float v0 = fmaf(g, wg.x, __builtin_ldexpf(acc[0][i], er - e0)), v1 = fmaf(g, wg.y, __builtin_ldexpf(acc[1][i], er - e1));
            if (t < A.T) {
                const size_t o = (size_t)t * kRgD + n0 + 2 * c;
                if constexpr (XF == Q36MOE_FMT_F32) *reinterpret_cast<float2 *>(static_cast<float *>(A.dx) + o) = make_float2(v0, v1);
                else *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(A.dx) + o) = bf16_pair(v0, v1);
            }
        }
    }
}

constexpr int kCUs = 256;
constexpr int kSplitT = 512;      // tokens from which the split operands pay

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
    if (T < kSplitT) return 1;
    const int span = dw_span(T, n_expert);
    return (T + span - 1) / span;
}

template <int XF>
void launch_product(const ProductArgs &P, float *dw, float *ws, hipStream_t s) {
    ProductArgs A = P;
    const bool many = A.T >= kSplitT;
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
    return nb == 1 ? 0 : (size_t)nb * (2 * n_expert + 1) * sizeof(float);
}

int q36moe_balance_loss(const float *logits, int ld, const int32_t *idx, const uint8_t *mask, int T, int n_expert, int k,
                        float coef, int32_t *counts, float *psum, float *loss, void *ws, size_t ws_bytes, void *stream) {
    if (T < 0 || n_expert < 1 || n_expert > kMaxE || ld < n_expert || k < 1 || k > kMaxK || k > n_expert)
        return Q36MOE_EINVAL;
    if (!counts || !psum || !loss || (T > 0 && (!logits || !idx))) return Q36MOE_EINVAL;
    const size_t need = q36moe_balance_loss_workspace(T, n_expert);
    if (need && (!ws || ws_bytes < need)) return Q36MOE_EINVAL;
    BalanceArgs A{logits, idx, mask, ld, T, n_expert, k, 0, coef, counts, psum, loss, static_cast<float *>(ws)};
    const int nb = T ? balance_groups(T) : 1;
    A.chunk = (int)(((int64_t)T + nb - 1) / nb);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n_expert <= 64) hipLaunchKernelGGL(k_balance<4>, dim3(nb), dim3(64 * kBalW), 0, s, A);
    else hipLaunchKernelGGL(k_balance<16>, dim3(nb), dim3(64 * kBalW), 0, s, A);
    if (nb > 1) hipLaunchKernelGGL(k_balance_join, dim3(1), dim3(1024), 0, s, A, nb);
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
    if (n_expert <= 64) hipLaunchKernelGGL(k_logit_grad<4>, g, dim3(256), 0, s, A);
    else hipLaunchKernelGGL(k_logit_grad<16>, g, dim3(256), 0, s, A);
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
        n_rows > kMaxRouterRows || ld < n_expert || (x_fmt != Q36MOE_FMT_F32 && x_fmt != Q36MOE_FMT_BF16) || (!dw && !dx) ||
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
    if (need && (!ws || ws_bytes < need)) return Q36MOE_EINVAL;
    ProductArgs A{};
    A.w = w; A.dl = dlogits; A.dsh = dshg; A.x = x; A.dx = dx;
    A.ld = ld; A.ld_sh = ld_shg ? ld_shg : 1;
    A.n_rows = n_rows; A.n_expert = n_expert; A.T = T;
    if (x_fmt == Q36MOE_FMT_F32) launch_product<Q36MOE_FMT_F32>(A, dw, static_cast<float *>(ws), s);
    else launch_product<Q36MOE_FMT_BF16>(A, dw, static_cast<float *>(ws), s);
    return hip_status(hipGetLastError());
}

}  // extern "C"
