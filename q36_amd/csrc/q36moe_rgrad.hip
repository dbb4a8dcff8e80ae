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
// gradients of the router product, fp32 on the matrix cores
// ---------------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kRgD = 2048;

struct ProductArgs {
    const float *w, *dl, *dsh;   // [n_rows][kRgD]; [T][ld]; the shared gate's column, stride ld_sh
    const void *x;
    float *dw;                   // [splits][n_rows][kRgD]
    void *dx;
    int ld, ld_sh, n_rows, n_expert, T, span;   // tokens per split
};

// v_mfma_f32_32x32x2_f32: lane L holds row (A) or column (B) L % 32 at K
// element L / 32; of C rows 8 (i / 4) + 4 (L / 32) + i % 4 of column L % 32.
__device__ __forceinline__ f32x16 mfma2(float a, float b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ int c_row(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

// dW: 32 router rows x 64 columns per wave, summed over the split's tokens.
// Both operands are read as they lie, 32 neighbouring values per half wave.
template <int XF>
__global__ __launch_bounds__(256) void k_router_dw(ProductArgs A) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int d0 = blockIdx.x * 256 + (threadIdx.x >> 6) * 64 + (lane & 31);
    const int r = min((int)blockIdx.y * 32 + (lane & 31), A.n_rows - 1);
    const bool sh = r >= A.n_expert;
    const float *col = sh ? A.dsh : A.dl + r;
    const int64_t step = sh ? A.ld_sh : A.ld;
    const int64_t t0 = (int64_t)blockIdx.z * A.span, t1 = min(t0 + A.span, (int64_t)A.T);
    f32x16 c0 = {}, c1 = {};
    constexpr int U = 8;
    for (int64_t t = t0; t < t1; t += 2 * U) {
        float a[U], b0[1], b1[U], b[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t tt = t + 2 * u + half;
            const int64_t tc = min(tt, t1 - 1);
            const bool in = tt < t1;
            a[u] = col[tc * step];
            load_row<XF>(A.x, (size_t)tc * kRgD + d0, b0);
            b[u] = in ? b0[0] : 0.0f;
            load_row<XF>(A.x, (size_t)tc * kRgD + d0 + 32, b0);
            b1[u] = in ? b0[0] : 0.0f;
            a[u] = in ? a[u] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            c0 = mfma2(a[u], b[u], c0);
            c1 = mfma2(a[u], b1[u], c1);
        }
    }
    float *o = A.dw + (size_t)blockIdx.z * A.n_rows * kRgD;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int row = blockIdx.y * 32 + c_row(i, lane);
        if (row < A.n_rows) {
            o[(size_t)row * kRgD + d0] = c0[i];
            o[(size_t)row * kRgD + d0 + 32] = c1[i];
        }
    }
}

// dx: 32 tokens x 64 columns per wave.  Lane half h of a step of 8 rows holds
// rows 4h..4h+3 of both operands.
template <int XF>
__global__ __launch_bounds__(256) void k_router_dx(ProductArgs A) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int64_t tb = (int64_t)(blockIdx.x / (kRgD / 256)) * 32;
    const int d0 = (blockIdx.x % (kRgD / 256)) * 256 + (threadIdx.x >> 6) * 64 + (lane & 31);
    const int64_t t = min(tb + (lane & 31), (int64_t)A.T - 1);
    const float *row = A.dl + (size_t)t * A.ld;
    f32x16 c0 = {}, c1 = {};
    const int whole = A.n_expert & ~7;
    int r0 = 0;
    for (; r0 < whole; r0 += 8) {
        const int r = r0 + 4 * half;
        float a[4];
        load_row<Q36MOE_FMT_F32>(row, r, a);
        float b0[4], b1[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            b0[i] = A.w[(size_t)(r + i) * kRgD + d0];
            b1[i] = A.w[(size_t)(r + i) * kRgD + d0 + 32];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c0 = mfma2(a[i], b0[i], c0);
            c1 = mfma2(a[i], b1[i], c1);
        }
    }
    // the rows left over, the shared gate's among them
    for (; r0 < A.n_rows; r0 += 2) {
        const int r = min(r0 + half, A.n_rows - 1);
        const bool in = r0 + half < A.n_rows;
        const float v = r < A.n_expert ? row[r] : A.dsh[t * A.ld_sh];
        const float a = in ? v : 0.0f;
        c0 = mfma2(a, in ? A.w[(size_t)r * kRgD + d0] : 0.0f, c0);
        c1 = mfma2(a, in ? A.w[(size_t)r * kRgD + d0 + 32] : 0.0f, c1);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int64_t tt = tb + c_row(i, lane);
        if (tt < A.T) {
            store_one<XF>(A.dx, (size_t)tt * kRgD + d0, c0[i]);
            store_one<XF>(A.dx, (size_t)tt * kRgD + d0 + 32, c1[i]);
        }
    }
}

constexpr int kMaxRouterT = 1 << 25;

// Splits of the tokens: enough waves to fill the chip.
int dw_splits(int T, int n_rows) {
    const int tiles = 8 * ((n_rows + 31) / 32);   // workgroups of one split
    const int want = (512 + tiles - 1) / tiles, most = (T + 127) / 128;
    return want < most ? want : most < 1 ? 1 : most;
}

template <int XF>
void launch_product(const ProductArgs &P, float *dw, float *ws, hipStream_t s) {
    ProductArgs A = P;
    if (dw) {
        const int splits = dw_splits(A.T, A.n_rows);
        A.span = (A.T + splits - 1) / splits;
        A.dw = splits == 1 ? dw : ws;
        hipLaunchKernelGGL(k_router_dw<XF>, dim3(kRgD / 256, (A.n_rows + 31) / 32, splits), dim3(256), 0, s, A);
        if (splits > 1) sum_partials(ws, splits, (size_t)A.n_rows * kRgD, (size_t)A.n_rows * kRgD, dw, nullptr, s);
    }
    if (A.dx)
        hipLaunchKernelGGL(k_router_dx<XF>, dim3((unsigned)((A.T + 31) / 32 * (kRgD / 256))), dim3(256), 0, s, A);
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
    const int n = dw_splits(T, n_rows);
    return n == 1 ? 0 : (size_t)n * n_rows * kRgD * sizeof(float);
}

int q36moe_router_logits_backward(const float *w, int n_rows, int n_expert, const void *x, int x_fmt, int T, int d_model,
                                  const float *dlogits, int ld, const float *dshg, int ld_shg, float *dw, void *dx, void *ws,
                                  size_t ws_bytes, void *stream) {
    if (T < 0 || T > kMaxRouterT || d_model != kRgD || n_expert < 1 || n_rows < n_expert || n_rows > n_expert + 1 ||
        n_rows > 65535 * 32 || ld < n_expert || (x_fmt != Q36MOE_FMT_F32 && x_fmt != Q36MOE_FMT_BF16) || (!dw && !dx) ||
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
    A.ld = ld; A.ld_sh = ld_shg ? ld_shg : 1; A.n_rows = n_rows; A.n_expert = n_expert; A.T = T;
    if (x_fmt == Q36MOE_FMT_F32) launch_product<Q36MOE_FMT_F32>(A, dw, static_cast<float *>(ws), s);
    else launch_product<Q36MOE_FMT_BF16>(A, dw, static_cast<float *>(ws), s);
    return hip_status(hipGetLastError());
}

}  // extern "C"
