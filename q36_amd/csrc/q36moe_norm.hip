// Layer norm and RMS norm in front of the MoE layer, forward (with the
// residual add) and backward (with the residual stream's gradient and the
// sums over tokens for weight and bias).
//
// Forward, per row:   v = x + a,  d = v - mean(v) (RMS norm: d = v),
//                     r = 1 / sqrt(mean(d^2) + eps),  y = d * r * w + b
// Backward, n = d * r, g = dy * w:
//                     dx = r * (g - mean(g) - n * mean(g * n)) + dres
//                     (RMS norm: without mean(g))
//                     dw = sum_t dy * n,  db = sum_t dy
// Both move each value once and are bound by memory: a row stays in the
// registers of the threads that loaded it from its statistics to its output.
#include "q36moe_rows.h"

namespace {

constexpr int kMaxNormD = 16384;

struct NormArgs {
    const void *x, *a;         // forward: x and addend; backward: h and dres
    const void *dy;
    void *h, *y;               // forward: sum and norm; backward: y is dx
    const float *w, *b;
    float *pw, *pb;            // backward: partial sums, a row of `pstride` floats per stream
    size_t pstride;
    int64_t ld_x, ld_a, ld_dy, ld_h, ld_y;
    int T, D, rms;
    int streams;               // backward
    float eps, inv_d;
};

// Sums of N values over the row's threads: a wave's own sum, or, with NW waves
// per row, the waves' sums through LDS in wave order.  `p` alternates between
// two buffers, so one barrier per sum separates a buffer's readers from its
// next writers.
template <int NW, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float (*red)[N * NW], int &p) {
#pragma unroll
    for (int i = 0; i < N; i++) s[i] = sum64(s[i]);
    if constexpr (NW > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) red[p][i * NW + wave] = s[i];
        lds_barrier();
#pragma unroll
        for (int i = 0; i < N; i++) {
            s[i] = red[p][i * NW];
#pragma unroll
            for (int k = 1; k < NW; k++) s[i] += red[p][i * NW + k];
        }
        p ^= 1;
    }
}

// 1 / sqrt(variance + eps); rounding may leave a variance just under 0, a NaN
// stays one.
__device__ __forceinline__ float inv_dev(float var, float eps) { return rsqrtf((var < 0.0f ? 0.0f : var) + eps); }

// A thread's vectors of a row: vector j holds columns col..col+VEC-1.  The
// row's last vector may reach past its end and vectors beyond it lie outside;
// both load the row's last VEC columns instead (no access leaves the row) and
// leave the first `skip` of them to the vectors they belong to.
template <int VEC, int TPR>
struct Cols {
    int at, skip;
    __device__ __forceinline__ Cols(int j, int tid, int D) {
        const int col = (j * TPR + tid) * VEC;
        at = min(col, D - VEC);
        skip = min(col - at, VEC);
    }
};

// One row per workgroup of NW waves (four rows of a wave each where NW is 1).
// Measured with residual: 4006 bf16 rows of 2048 13 us (5.0 TB/s), 16384 fp32 rows
// 94 us (5.7 TB/s); 4096 fp32 rows with bf16 y by 1 / 2 / 4 waves 28 / 25 / 24 us.
template <int XF, int YF, int VEC, int NW, int NV>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void k_layernorm(NormArgs A) {
    constexpr int TPR = 64 * NW, RPB = NW == 1 ? 4 : 1;
    __shared__ float red1[2][NW], red2[2][2 * NW];
    const int tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
    int p1 = 0, p2 = 0;
    for (int64_t t = (int64_t)blockIdx.x * RPB + (NW == 1 ? threadIdx.x >> 6 : 0); t < A.T; t += (int64_t)gridDim.x * RPB) {
        float v[NV][VEC];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const Cols<VEC, TPR> c(j, tid, A.D);
            load_row<XF>(A.x, t * A.ld_x + c.at, v[j]);
        }
        if (A.a) {
            float a[NV][VEC];
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const Cols<VEC, TPR> c(j, tid, A.D);
                load_row<XF>(A.a, t * A.ld_a + c.at, a[j]);
            }
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int i = 0; i < VEC; i++) v[j][i] += a[j][i];
        }
        // the mean first, then the squares about it; the second pass also sums
        // the deviations, which corrects the rounding of the mean in rows whose
        // offset is many times their spread
        float m0 = 0.0f;
        if (!A.rms) {
            float s[1] = {0.0f};
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const Cols<VEC, TPR> c(j, tid, A.D);
#pragma unroll
                for (int i = 0; i < VEC; i++) s[0] += i >= c.skip ? v[j][i] : 0.0f;
            }
            row_sums<NW>(s, red1, p1);
            m0 = s[0] * A.inv_d;
        }
        float q[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const Cols<VEC, TPR> c(j, tid, A.D);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = i >= c.skip ? v[j][i] - m0 : 0.0f;
                q[0] += d;
                q[1] = fmaf(d, d, q[1]);
            }
        }
        row_sums<NW>(q, red2, p2);
        const float m1 = A.rms ? 0.0f : q[0] * A.inv_d;
        const float r = inv_dev(q[1] * A.inv_d - m1 * m1, A.eps);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const Cols<VEC, TPR> c(j, tid, A.D);
            if (c.skip < VEC) {
                float w[VEC], b[VEC], y[VEC];
#pragma unroll
                for (int i = 0; i < VEC; i++) { w[i] = 1.0f; b[i] = 0.0f; }
                if (A.w) load_row<Q36MOE_FMT_F32>(A.w, c.at, w);
                if (A.b) load_row<Q36MOE_FMT_F32>(A.b, c.at, b);
#pragma unroll
                for (int i = 0; i < VEC; i++) y[i] = fmaf(((v[j][i] - m0) - m1) * r, w[i], b[i]);
                if (A.h) store_row<XF>(A.h, t * A.ld_h + c.at, v[j], c.skip);
                store_row<YF>(A.y, t * A.ld_y + c.at, y, c.skip);
            }
        }
    }
}

// Streams (a workgroup, or a wave where NW is 1) take rows in turn and keep
// their columns' sums for weight and bias in registers; each leaves one row of
// partial sums.
template <int XF, int YF, int VEC, int NW, int NV>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void k_layernorm_backward(NormArgs A) {
    constexpr int TPR = 64 * NW, RPB = NW == 1 ? 4 : 1;
    __shared__ float red1[2][NW], red4[2][4 * NW];
    const int tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int stream = blockIdx.x * RPB + (NW == 1 ? threadIdx.x >> 6 : 0);
    int p1 = 0, p4 = 0;
    float sw[NV][VEC], sb[NV][VEC], w[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; j++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            sw[j][i] = sb[j][i] = 0.0f;
            w[j][i] = 1.0f;
        }
        if (A.w) load_row<Q36MOE_FMT_F32>(A.w, Cols<VEC, TPR>(j, tid, A.D).at, w[j]);
    }
    // a row's loads are made before the sums of the row before it (past the last
    // row it is read again), where registers allow
    constexpr bool AHEAD = NV * VEC <= 16;
    Bits<XF, VEC> bx[NV], ba[NV];
    Bits<YF, VEC> bg[NV];
    auto load = [&](int64_t t) {
        t = min(t, (int64_t)A.T - 1);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const Cols<VEC, TPR> c(j, tid, A.D);
            bx[j].load(A.x, t * A.ld_x + c.at);
            bg[j].load(A.dy, t * A.ld_dy + c.at);
        }
        if (A.a)
#pragma unroll
            for (int j = 0; j < NV; j++) ba[j].load(A.a, t * A.ld_a + Cols<VEC, TPR>(j, tid, A.D).at);
    };
    if (AHEAD) load(stream);
    const int64_t stride = (int64_t)gridDim.x * RPB;
    for (int64_t t = stream; t < A.T; t += stride) {
        float v[NV][VEC], g[NV][VEC];
        Bits<XF, VEC> res[NV];
        if (!AHEAD) load(t);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            res[j] = ba[j];
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                v[j][i] = bx[j][i];
                g[j][i] = bg[j][i];
            }
        }
        if (AHEAD) load(t + stride);
        float m0 = 0.0f;
        if (!A.rms) {
            float s[1] = {0.0f};
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const Cols<VEC, TPR> c(j, tid, A.D);
#pragma unroll
                for (int i = 0; i < VEC; i++) s[0] += i >= c.skip ? v[j][i] : 0.0f;
            }
            row_sums<NW>(s, red1, p1);
            m0 = s[0] * A.inv_d;
        }
        // sums of d, d^2, g and g * d over the row; dy of columns that belong to
        // another vector counts as 0
        float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const Cols<VEC, TPR> c(j, tid, A.D);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = i >= c.skip ? v[j][i] - m0 : 0.0f;
                g[j][i] = i >= c.skip ? g[j][i] : 0.0f;
                const float gw = g[j][i] * w[j][i];
                v[j][i] = d;
                q[0] += d;
                q[1] = fmaf(d, d, q[1]);
                q[2] += gw;
                q[3] = fmaf(gw, d, q[3]);
            }
        }
        row_sums<NW>(q, red4, p4);
        const float m1 = A.rms ? 0.0f : q[0] * A.inv_d;
        const float r = inv_dev(q[1] * A.inv_d - m1 * m1, A.eps);
        const float mg = A.rms ? 0.0f : q[2] * A.inv_d;
        const float mgn = (q[3] - m1 * q[2]) * r * A.inv_d;   // mean of g * n
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const Cols<VEC, TPR> c(j, tid, A.D);
            float o[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float n = (v[j][i] - m1) * r;
                sw[j][i] = fmaf(g[j][i], n, sw[j][i]);
                sb[j][i] += g[j][i];
                o[i] = (fmaf(g[j][i], w[j][i], -mg) - n * mgn) * r;
                if (A.a) o[i] += res[j][i];
            }
            if (A.y && c.skip < VEC) store_row<XF>(A.y, t * A.ld_y + c.at, o, c.skip);
        }
    }
    if (stream >= A.T) return;   // the last workgroup's waves past the last row have no partial row
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const Cols<VEC, TPR> c(j, tid, A.D);
        if (c.skip < VEC) {
            if (A.pw) store_row<Q36MOE_FMT_F32>(A.pw, stream * A.pstride + c.at, sw[j], c.skip);
            if (A.pb) store_row<Q36MOE_FMT_F32>(A.pb, stream * A.pstride + c.at, sb[j], c.skip);
        }
    }
}

// Rows of up to 512 columns go to one wave, longer ones to a workgroup of 4
// waves, past 4096 of 8: 4 to 16 values of each input per thread, 32 past 8192.
constexpr int kWaveRow = 512;
// Streams of the backward pass, each with a row of partial sums that is written
// and read again: a row of tokens each up to 256, then 4 rows and more.  256 of
// them (one workgroup per CU) have enough in flight where a row is 16 KiB and more,
// 512 below that: us at 16384 tokens with 256 / 512 / 1024 streams, 2048 columns
// fp32 97 / 102 / 112, bf16 77 / 58 / 63, 4096 columns fp32 with bf16 dy
// 174 / 183 / 190 (without the loads ahead 292 / 198 / 220).  Past 256 a multiple of
// 4: the four waves of a workgroup are streams where NW is 1, and each has rows.
constexpr int kMaxStreams = 512;

int streams(int T, size_t row_bytes) {
    const int most = row_bytes >= 16384 ? kMaxStreams / 2 : kMaxStreams;
    if (T <= kMaxStreams / 2) return T;
    const int n = (int)(((int64_t)T + 15) / 16) * 4;
    return n < kMaxStreams / 2 ? kMaxStreams / 2 : n < most ? n : most;
}

template <bool BWD, int XF, int YF, int VEC, int NW, int NV>
void launch_norm(const NormArgs &A, hipStream_t s) {
    constexpr int RPB = NW == 1 ? 4 : 1;
    if constexpr (BWD)
        hipLaunchKernelGGL((k_layernorm_backward<XF, YF, VEC, NW, NV>), dim3((A.streams + RPB - 1) / RPB),
                           dim3(NW == 1 ? 256 : 64 * NW), 0, s, A);
    else
        hipLaunchKernelGGL((k_layernorm<XF, YF, VEC, NW, NV>), dim3(((A.T < (1 << 20) ? A.T : (1 << 20)) + RPB - 1) / RPB),
                           dim3(NW == 1 ? 256 : 64 * NW), 0, s, A);
}

template <bool BWD, int XF, int YF>
void norm_by_width(const NormArgs &A, hipStream_t s) {
    constexpr int B = XF == Q36MOE_FMT_BF16 && YF == Q36MOE_FMT_BF16 ? 2 : 1;   // 16-byte vectors
    constexpr int VEC = 4 * B;
    const int D = A.D;
    if (D < VEC) launch_norm<BWD, XF, YF, 1, 1, 1>(A, s);
    else if (D <= 256 * B) launch_norm<BWD, XF, YF, VEC, 1, 1>(A, s);
    else if (D <= kWaveRow) launch_norm<BWD, XF, YF, VEC, 1, 2 / B>(A, s);
    else if (D <= 1024 * B) launch_norm<BWD, XF, YF, VEC, 4, 1>(A, s);
    else if (D <= 2048 * B) launch_norm<BWD, XF, YF, VEC, 4, 2>(A, s);
    else if (D <= 4096 * B) launch_norm<BWD, XF, YF, VEC, 4, 4>(A, s);
    else if (D <= 8192) launch_norm<BWD, XF, YF, VEC, 8, 4 / B>(A, s);
    else launch_norm<BWD, XF, YF, VEC, 8, 8 / B>(A, s);
}

template <bool BWD>
void norm_by_format(const NormArgs &A, int xf, int yf, hipStream_t s) {
    if (xf == Q36MOE_FMT_F32) {
        if (yf == Q36MOE_FMT_F32) norm_by_width<BWD, Q36MOE_FMT_F32, Q36MOE_FMT_F32>(A, s);
        else norm_by_width<BWD, Q36MOE_FMT_F32, Q36MOE_FMT_BF16>(A, s);
    } else {
        if (yf == Q36MOE_FMT_F32) norm_by_width<BWD, Q36MOE_FMT_BF16, Q36MOE_FMT_F32>(A, s);
        else norm_by_width<BWD, Q36MOE_FMT_BF16, Q36MOE_FMT_BF16>(A, s);
    }
}

bool fmt_ok(int f) { return f == Q36MOE_FMT_F32 || f == Q36MOE_FMT_BF16; }

bool norm_ok(int T, int D, float eps, int kind, int xf, int yf) {
    return T >= 0 && D >= 1 && D <= kMaxNormD && eps >= 0.0f && eps <= 3.40282347e38f &&
           (kind == Q36MOE_NORM_LAYER || kind == Q36MOE_NORM_RMS) && fmt_ok(xf) && fmt_ok(yf);
}

}  // namespace

extern "C" {

int q36moe_layernorm(const void *x, int64_t ld_x, const void *a, int64_t ld_a, int x_fmt, const float *w, const float *b,
                     int T, int d_model, float eps, int kind, void *h, int64_t ld_h, void *y, int64_t ld_y, int y_fmt,
                     void *stream) {
    if (!norm_ok(T, d_model, eps, kind, x_fmt, y_fmt) || ld_x < d_model || ld_y < d_model || (!a) != (!h) ||
        (a && (ld_a < d_model || ld_h < d_model)))
        return Q36MOE_EINVAL;
    if (T == 0) return Q36MOE_OK;
    if (!x || !y) return Q36MOE_EINVAL;
    NormArgs A{};
    A.x = x; A.a = a; A.h = h; A.y = y; A.w = w; A.b = b;
    A.ld_x = ld_x; A.ld_a = ld_a; A.ld_h = ld_h; A.ld_y = ld_y;
    A.T = T; A.D = d_model; A.rms = kind == Q36MOE_NORM_RMS; A.eps = eps; A.inv_d = 1.0f / (float)d_model;
    norm_by_format<false>(A, x_fmt, y_fmt, static_cast<hipStream_t>(stream));
    return hip_status(hipGetLastError());
}

size_t q36moe_layernorm_backward_workspace(int T, int d_model) {
    if (T < 2 || d_model < 1 || d_model > kMaxNormD) return 0;
    return (size_t)streams(T, 0) * 2 * d_model * sizeof(float);   // the most, whatever the formats
}

int q36moe_layernorm_backward(const void *dy, int64_t ld_dy, int y_fmt, const void *h, int64_t ld_h, const void *dres,
                              int64_t ld_dres, int x_fmt, const float *w, int T, int d_model, float eps, int kind, void *dx,
                              int64_t ld_dx, float *dw, float *db, void *ws, size_t ws_bytes, void *stream) {
    if (!norm_ok(T, d_model, eps, kind, x_fmt, y_fmt) || ld_dy < d_model || ld_h < d_model || (!dx && !dw && !db) ||
        (dx && ld_dx < d_model) || (dres && (!dx || ld_dres < d_model)))
        return Q36MOE_EINVAL;
    const bool sums = dw || db;
    if (T == 0 && !sums) return Q36MOE_OK;
    if (T > 0 && (!dy || !h)) return Q36MOE_EINVAL;
    if (sums && !workspace_ok(ws, ws_bytes, q36moe_layernorm_backward_workspace(T, d_model))) return Q36MOE_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const size_t D = (size_t)d_model;
    const size_t L = D * ((dw ? 1 : 0) + (db ? 1 : 0));
    const int xb = x_fmt == Q36MOE_FMT_F32 ? 4 : 2, yb = y_fmt == Q36MOE_FMT_F32 ? 4 : 2;
    const int n = streams(T, D * (2 * xb + yb));
    if (T > 0) {
        NormArgs A{};
        A.x = h; A.a = dres; A.dy = dy; A.y = dx; A.w = w;
        A.ld_x = ld_h; A.ld_a = ld_dres; A.ld_dy = ld_dy; A.ld_y = ld_dx;
        A.T = T; A.D = d_model; A.rms = kind == Q36MOE_NORM_RMS; A.eps = eps; A.inv_d = 1.0f / (float)d_model;
        A.pstride = L;
        A.streams = n;
        float *p = static_cast<float *>(ws);
        A.pw = !dw ? nullptr : T == 1 ? dw : p;   // one stream's partial row is the sum
        A.pb = !db ? nullptr : T == 1 ? db : p + (dw ? D : 0);
        norm_by_format<true>(A, x_fmt, y_fmt, s);
    }
    // no tokens: sums of nothing
    if (sums && T != 1) sum_partials(static_cast<const float *>(ws), n, L, dw ? D : 0, dw, db, s);
    return hip_status(hipGetLastError());
}

}  // extern "C"
