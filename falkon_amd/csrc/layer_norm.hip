// Layer norm of the rows of a matrix and its backward pass (gfx950).
//
//   y  = (x - mean) * rstd * w + b,     mean = sum(x) / d,  rstd = 1 / sqrt(sum((x - mean)^2) / d + eps)
//   dx = rstd * (g - sum(g)/d - z * sum(g z)/d),   g = dy * w,  z = (x - mean) * rstd
//   dw = sum over rows of dy * z,   db = sum over rows of dy
//
// Both passes move every value once and are bound by memory.  A row lies in the registers of `TPR` threads (NV vectors
// of 16 bytes each), so mean and centred sum of squares are two passes over registers, not over memory, and nothing
// cancels as it does in sum(x^2) - mean^2.  Sums are held in 32 bits (64 for double).  What that leaves in the mean, a few units of its
// last digit, is the same for all values of a row (a row of 784 times 10000.1 would come out as -0.3): it is the mean of the centred
// values r, so the second pass sums them too, takes c = sum(r) / d from each and c^2 from the variance.  The backward pass, whose z start
// from the rounded mean, does the same with the mean of z.  Short rows share a wave (28
// floats: eight threads a row), rows of more than kRowThreads * 8 vectors are read again instead of being kept.
// In the backward pass a workgroup walks over many rows and keeps its share of dw and db in registers; it writes one
// partial row at its end, and a second kernel adds those in a fixed order: no atomics, results are the same run to run.
#include "flk_common.h"
#include "element_types.h"

namespace flk {

constexpr int kRowThreads = 256;
constexpr int kLoopThreads = 1024;

template <typename T> struct NormAcc { typedef float type; };
template <> struct NormAcc<double> { typedef double type; };

__device__ __forceinline__ float rsqrt_of(float x) { return 1.0f / sqrtf(x); }
__device__ __forceinline__ double rsqrt_of(double x) { return 1.0 / sqrt(x); }

// (16 bytes are what the callers see to: eight float weights beside eight 16-bit values are two such)
template <typename T, int VEC> struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) NormVec { T v[VEC]; };

// `VEC` consecutive values from element i of a row on, converted; past `d` zero
template <typename T, int VEC, typename A>
__device__ __forceinline__ void load_vec(const T *p, int64_t i, int64_t d, A *r) {
    if (i < d) {
        const NormVec<T, VEC> t = *reinterpret_cast<const NormVec<T, VEC> *>(p + i);
#pragma unroll
        for (int j = 0; j < VEC; j++) r[j] = to_acc<A>(t.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) r[j] = A(0);
    }
}
template <typename T, int VEC, typename A>
__device__ __forceinline__ void store_vec(T *p, int64_t i, int64_t d, const A *r) {
    if (i >= d) return;
    NormVec<T, VEC> t;
#pragma unroll
    for (int j = 0; j < VEC; j++) t.v[j] = from_acc<T>(r[j]);
    *reinterpret_cast<NormVec<T, VEC> *>(p + i) = t;
}
// weights come in the data's type or in float
template <typename T, int VEC, typename A>
__device__ __forceinline__ void load_weight(const void *w, int wide, int64_t i, int64_t d, A *r) {
    if (wide) load_vec<float, VEC, A>((const float *)w, i, d, r);
    else load_vec<T, VEC, A>((const T *)w, i, d, r);
}

// Sum over the TPR threads that share a row; every one of them gets it.  Fixed order.
template <int TPR, typename A>
__device__ __forceinline__ A row_sum(A x, A *lds) {
#pragma unroll
    for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();                         // the previous sum may still be being read
        if ((threadIdx.x & 63) == 0) lds[wave] = x;
        __syncthreads();
        x = A(0);
#pragma unroll
        for (int w = 0; w < TPR / 64; w++) x += lds[w];
    }
    return x;
}

// N sums at once; with several waves a row one barrier suffices if another stands between this call's reads and the next one's writes
// (the caller alternates between two places in LDS, or sums something else in between).
template <int TPR, int N, typename A>
__device__ __forceinline__ void row_sums(A (&x)[N], A *lds) {
#pragma unroll
    for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) x[i] += __shfl_xor(x[i], off, 64);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; i++) lds[N * wave + i] = x[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            x[i] = A(0);
#pragma unroll
            for (int w = 0; w < TPR / 64; w++) x[i] += lds[N * w + i];
        }
    }
}
// The correction c of a rounded mean, and the variance, from the sums of the centred values and of their squares
template <typename A> __device__ __forceinline__ A centre(const A (&sums)[2], A inv_d, A &var) {
    const A c = sums[0] * inv_d;
    var = sums[1] * inv_d - c * c;
    var = var < A(0) ? A(0) : var;                                 // (NaN stays NaN)
    return c;
}

template <typename T> struct NormArgs {
    typedef typename NormAcc<T>::type acc;
    const T *x, *dy;
    T *y;                  // forward: y, backward: dx
    const void *w, *b;
    acc *mean, *rstd;
    acc *partial;          // backward: [workgroups][2][d]
    acc *shift;            // backward, long rows: the mean of z, [rows]
    int64_t rows, d, x_rs, dy_rs;
    int wide;              // w and b are float
    double eps;
};

template <typename T, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(kRowThreads) layer_norm_kernel(NormArgs<T> p) {
    typedef typename NormArgs<T>::acc A;
    constexpr int kRows = kRowThreads / TPR;
    __shared__ A lds[3 * kRowThreads / 64];
    const int sub = threadIdx.x % TPR;
    const A inv_d = A(1) / A(p.d);
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < p.rows; row0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = row0 + threadIdx.x / TPR;
        const bool live = row < p.rows;
        const T *x = p.x + (live ? row : p.rows - 1) * p.x_rs;
        A r[NV][VEC];
        A s = A(0);
#pragma unroll
        for (int n = 0; n < NV; n++) {
            load_vec<T, VEC, A>(x, (int64_t)(n * TPR + sub) * VEC, p.d, r[n]);
#pragma unroll
            for (int j = 0; j < VEC; j++) s += r[n][j];
        }
        const A mean = row_sum<TPR, A>(s, lds) * inv_d;
        A sums[2] = {A(0), A(0)}, var;
#pragma unroll
        for (int n = 0; n < NV; n++) {
            if ((int64_t)(n * TPR + sub) * VEC < p.d) {
#pragma unroll
                for (int j = 0; j < VEC; j++) { r[n][j] -= mean; sums[0] += r[n][j]; sums[1] += r[n][j] * r[n][j]; }
            }
        }
        row_sums<TPR, 2, A>(sums, lds + kRowThreads / 64);
        const A c = centre(sums, inv_d, var), rstd = rsqrt_of(var + A(p.eps));
        if (!live) continue;
        if (sub == 0 && p.mean != nullptr) { p.mean[row] = mean + c; p.rstd[row] = rstd; }
#pragma unroll
        for (int n = 0; n < NV; n++)
#pragma unroll
            for (int j = 0; j < VEC; j++) r[n][j] -= c;
#pragma unroll
        for (int n = 0; n < NV; n++) {
            const int64_t i = (int64_t)(n * TPR + sub) * VEC;
            A w[VEC], b[VEC];
            if (p.w != nullptr) {
                load_weight<T, VEC, A>(p.w, p.wide, i, p.d, w);
#pragma unroll
                for (int j = 0; j < VEC; j++) r[n][j] *= rstd * w[j];
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j++) r[n][j] *= rstd;
            }
            if (p.b != nullptr) {
                load_weight<T, VEC, A>(p.b, p.wide, i, p.d, b);
#pragma unroll
                for (int j = 0; j < VEC; j++) r[n][j] += b[j];
            }
            store_vec<T, VEC, A>(p.y + row * p.d, i, p.d, r[n]);
        }
    }
}

// Rows too long for the registers: read three times, the later ones from the caches.
template <typename T>
__global__ void __launch_bounds__(kLoopThreads) layer_norm_long_kernel(NormArgs<T> p) {
    typedef typename NormArgs<T>::acc A;
    __shared__ A lds[3 * kLoopThreads / 64];
    const A inv_d = A(1) / A(p.d);
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *x = p.x + row * p.x_rs;
        A s = A(0);
        for (int64_t i = threadIdx.x; i < p.d; i += kLoopThreads) s += to_acc<A>(x[i]);
        const A mean = row_sum<kLoopThreads, A>(s, lds) * inv_d;
        A sums[2] = {A(0), A(0)}, var;
        for (int64_t i = threadIdx.x; i < p.d; i += kLoopThreads) { const A r = to_acc<A>(x[i]) - mean; sums[0] += r; sums[1] += r * r; }
        row_sums<kLoopThreads, 2, A>(sums, lds + kLoopThreads / 64);
        const A c = centre(sums, inv_d, var), rstd = rsqrt_of(var + A(p.eps));
        if (threadIdx.x == 0 && p.mean != nullptr) { p.mean[row] = mean + c; p.rstd[row] = rstd; }
        for (int64_t i = threadIdx.x; i < p.d; i += kLoopThreads) {
            A w = A(1), b = A(0);
            if (p.w != nullptr) load_weight<T, 1, A>(p.w, p.wide, i, p.d, &w);
            if (p.b != nullptr) load_weight<T, 1, A>(p.b, p.wide, i, p.d, &b);
            p.y[row * p.d + i] = from_acc<T>((to_acc<A>(x[i]) - mean - c) * (rstd * w) + b);
        }
    }
}

template <typename T, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(kRowThreads) layer_norm_bwd_kernel(NormArgs<T> p) {
    typedef typename NormArgs<T>::acc A;
    constexpr int kRows = kRowThreads / TPR;
    constexpr int kWidth = TPR * NV * VEC;             // columns a row's threads hold
    constexpr int kLds = TPR <= 64 ? 2 * kWidth : 6 * (kRowThreads / 64);
    __shared__ A lds[kLds];
    const int sub = threadIdx.x % TPR;
    const A inv_d = A(1) / A(p.d);
    A dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int n = 0; n < NV; n++)
#pragma unroll
        for (int j = 0; j < VEC; j++) dw[n][j] = db[n][j] = A(0);
    // the next row's values are on their way while the present one's are summed
    NormVec<T, VEC> nx[NV], ny[NV];
    A n_mean = A(0), n_rstd = A(0);
    const auto fetch = [&](int64_t row0) {
        const int64_t row = row0 + threadIdx.x / TPR, at = row < p.rows ? row : p.rows - 1;
        n_mean = p.mean[at];
        n_rstd = p.rstd[at];
#pragma unroll
        for (int n = 0; n < NV; n++) {
            const int64_t i = (int64_t)(n * TPR + sub) * VEC;
            if (i < p.d) {
                nx[n] = *reinterpret_cast<const NormVec<T, VEC> *>(p.x + at * p.x_rs + i);
                ny[n] = *reinterpret_cast<const NormVec<T, VEC> *>(p.dy + at * p.dy_rs + i);
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * kRows;
    int64_t row0 = (int64_t)blockIdx.x * kRows;
    if (row0 < p.rows) fetch(row0);
    for (int turn = 0; row0 < p.rows; row0 += step, turn ^= 1) {
        const int64_t row = row0 + threadIdx.x / TPR;
        const bool live = row < p.rows;
        const A mean = n_mean, rstd = n_rstd;
        A z[NV][VEC], g[NV][VEC];
        NormVec<T, VEC> dy[NV];
        A sums[3] = {A(0), A(0), A(0)};                            // of g, g z and z
#pragma unroll
        for (int n = 0; n < NV; n++) {
            const int64_t i = (int64_t)(n * TPR + sub) * VEC;
            dy[n] = ny[n];
            A w[VEC];
            if (p.w != nullptr) load_weight<T, VEC, A>(p.w, p.wide, i, p.d, w);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                z[n][j] = i < p.d ? (to_acc<A>(nx[n].v[j]) - mean) * rstd : A(0);
                g[n][j] = i < p.d ? to_acc<A>(ny[n].v[j]) : A(0);
                if (p.w != nullptr) g[n][j] *= w[j];
                sums[0] += g[n][j];
                sums[1] += g[n][j] * z[n][j];
                sums[2] += z[n][j];
            }
        }
        if (row0 + step < p.rows) fetch(row0 + step);
        row_sums<TPR, 3, A>(sums, lds + (TPR > 64 ? turn * 3 * (kRowThreads / 64) : 0));
        const A c = sums[2] * inv_d, s1 = sums[0] * inv_d, s2 = sums[1] * inv_d - c * s1;
        if (!live) continue;
#pragma unroll
        for (int n = 0; n < NV; n++) {
            const int64_t i = (int64_t)(n * TPR + sub) * VEC;
            if (i < p.d) {
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    z[n][j] -= c;
                    const A t = to_acc<A>(dy[n].v[j]);
                    dw[n][j] += t * z[n][j];
                    db[n][j] += t;
                }
            }
            if (p.y == nullptr) continue;
#pragma unroll
            for (int j = 0; j < VEC; j++) g[n][j] = rstd * (g[n][j] - s1 - z[n][j] * s2);
            store_vec<T, VEC, A>(p.y + row * p.d, i, p.d, g[n]);
        }
    }
    if (p.partial == nullptr) return;
    A *out = p.partial + (int64_t)blockIdx.x * 2 * p.d;
    if constexpr (TPR <= 64) {
        // rows of one wave first, then wave after wave through LDS
#pragma unroll
        for (int n = 0; n < NV; n++)
#pragma unroll
            for (int j = 0; j < VEC; j++)
#pragma unroll
                for (int off = TPR; off < 64; off <<= 1) {
                    dw[n][j] += __shfl_xor(dw[n][j], off, 64);
                    db[n][j] += __shfl_xor(db[n][j], off, 64);
                }
        for (int wave = 0; wave < kRowThreads / 64; wave++) {
            __syncthreads();
            if ((int)(threadIdx.x >> 6) == wave && (threadIdx.x & 63) < TPR) {
#pragma unroll
                for (int n = 0; n < NV; n++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const int c = (n * TPR + sub) * VEC + j;
                        lds[c] = (wave ? lds[c] : A(0)) + dw[n][j];
                        lds[kWidth + c] = (wave ? lds[kWidth + c] : A(0)) + db[n][j];
                    }
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < p.d; c += kRowThreads) { out[c] = lds[c]; out[p.d + c] = lds[kWidth + c]; }
    } else {
#pragma unroll
        for (int n = 0; n < NV; n++) {
            const int64_t i = (int64_t)(n * TPR + sub) * VEC;
            if (i < p.d) {
#pragma unroll
                for (int j = 0; j < VEC; j++) { out[i + j] = dw[n][j]; out[p.d + i + j] = db[n][j]; }
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kLoopThreads) layer_norm_bwd_long_kernel(NormArgs<T> p) {
    typedef typename NormArgs<T>::acc A;
    __shared__ A lds[2][3 * kLoopThreads / 64];
    const A inv_d = A(1) / A(p.d);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T *x = p.x + row * p.x_rs, *dy = p.dy + row * p.dy_rs;
        const A mean = p.mean[row], rstd = p.rstd[row];
        A sums[3] = {A(0), A(0), A(0)};                            // of g, g z and z
        for (int64_t i = threadIdx.x; i < p.d; i += kLoopThreads) {
            A w = A(1);
            if (p.w != nullptr) load_weight<T, 1, A>(p.w, p.wide, i, p.d, &w);
            const A g = to_acc<A>(dy[i]) * w, z = (to_acc<A>(x[i]) - mean) * rstd;
            sums[0] += g;
            sums[1] += g * z;
            sums[2] += z;
        }
        row_sums<kLoopThreads, 3, A>(sums, lds[turn]);
        const A c = sums[2] * inv_d, s1 = sums[0] * inv_d, s2 = sums[1] * inv_d - c * s1;
        if (threadIdx.x == 0 && p.shift != nullptr) p.shift[row] = c;
        if (p.y == nullptr) continue;
        for (int64_t i = threadIdx.x; i < p.d; i += kLoopThreads) {
            A w = A(1);
            if (p.w != nullptr) load_weight<T, 1, A>(p.w, p.wide, i, p.d, &w);
            const A z = (to_acc<A>(x[i]) - mean) * rstd - c;
            p.y[row * p.d + i] = from_acc<T>(rstd * (to_acc<A>(dy[i]) * w - s1 - z * s2));
        }
    }
}
// the long rows' share of dw and db: a thread owns a column, blockIdx.y a set of rows
template <typename T>
__global__ void __launch_bounds__(kRowThreads) layer_norm_columns_kernel(NormArgs<T> p) {
    typedef typename NormArgs<T>::acc A;
    const int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
    if (i >= p.d) return;
    A dw = A(0), db = A(0);
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const A g = to_acc<A>(p.dy[row * p.dy_rs + i]);
        dw += g * ((to_acc<A>(p.x[row * p.x_rs + i]) - p.mean[row]) * p.rstd[row] - p.shift[row]);
        db += g;
    }
    p.partial[(int64_t)blockIdx.y * 2 * p.d + i] = dw;
    p.partial[(int64_t)blockIdx.y * 2 * p.d + p.d + i] = db;
}

// dw[c] and db[c] from the workgroups' partial rows: 32 columns by 32 slices of the rows a workgroup
template <typename T, typename O>
__global__ void __launch_bounds__(1024) layer_norm_finish_kernel(const typename NormAcc<T>::type *partial, int parts, int64_t d,
                                                                 O *dw, O *db) {
    typedef typename NormAcc<T>::type A;
    __shared__ A lds[32][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + col;
    A s = A(0);
    if (c < 2 * d)
        for (int i = slice; i < parts; i += 32) s += partial[(int64_t)i * 2 * d + c];
    lds[slice][col] = s;
    __syncthreads();
    if (slice != 0 || c >= 2 * d) return;
    s = A(0);
#pragma unroll
    for (int i = 0; i < 32; i++) s += lds[i][col];
    if (c < d) { if (dw != nullptr) dw[c] = from_acc<O>(s); }
    else if (db != nullptr) db[c - d] = from_acc<O>(s);
}

// Row layouts: the fewest threads that hold a row, up to one vector each in a wave, then more vectors, then four waves.
// A workgroup's sums over its waves cost two barriers each, so rows stay in one wave as long as four vectors a thread do.
struct NormPlan { int vec, tpr, nv; };
template <typename T> inline NormPlan norm_plan(int64_t d, bool aligned) {
    const int vec = aligned ? 16 / (int)sizeof(T) : 1;
    const int64_t n = (d + vec - 1) / vec;
    if (n <= 8) return {vec, 8, 1};
    if (n <= 16) return {vec, 16, 1};
    if (n <= 32) return {vec, 32, 1};
    if (n <= 64) return {vec, 64, 1};
    if (n <= 128) return {vec, 64, 2};
    if (n <= 256) return {vec, 64, 4};
    if (n <= 512) return {vec, kRowThreads, 2};
    if (n <= 1024) return {vec, kRowThreads, 4};
    if (n <= 2048) return {vec, kRowThreads, 8};
    return {1, kLoopThreads, 0};
}
inline int64_t norm_min(int64_t a, int64_t b) { return a < b ? a : b; }
// Workgroups of the backward pass: as many partial rows are written and read again, so no more than are needed to fill
// the chip, and at least eight rows of a wave (or workgroup) each.
inline int64_t norm_bwd_groups(int64_t rows, const NormPlan &p) {
    const int64_t per = p.nv == 0 ? 1 : kRowThreads / p.tpr;
    const int64_t most = p.tpr <= 64 ? 1024 : 512;
    const int64_t n = (rows + 8 * per - 1) / (8 * per);
    return n < 1 ? 1 : norm_min(n, most);
}

#define FLK_NORM_PLANS(CALL)                                                             \
    if (plan.nv == 0) { CALL(0, 0) }                                                     \
    else if (plan.tpr == 8) { CALL(8, 1) } else if (plan.tpr == 16) { CALL(16, 1) }      \
    else if (plan.tpr == 32) { CALL(32, 1) }                                             \
    else if (plan.tpr == 64) { if (plan.nv == 1) { CALL(64, 1) } else if (plan.nv == 2) { CALL(64, 2) } else { CALL(64, 4) } } \
    else if (plan.nv == 2) { CALL(256, 2) } else if (plan.nv == 4) { CALL(256, 4) } else { CALL(256, 8) }

template <typename T, int VEC> void norm_forward(const NormArgs<T> &a, const NormPlan &plan, hipStream_t st) {
#define FLK_CALL(TPR, NV)                                                                                              \
    if constexpr (NV == 0) {                                                                                           \
        hipLaunchKernelGGL((layer_norm_long_kernel<T>), dim3((unsigned)norm_min(a.rows, 4096)), dim3(kLoopThreads), 0, st, a); \
    } else {                                                                                                           \
        const int64_t groups = (a.rows + kRowThreads / TPR - 1) / (kRowThreads / TPR);                                 \
        hipLaunchKernelGGL((layer_norm_kernel<T, VEC, TPR, NV>), dim3((unsigned)norm_min(groups, 16384)), dim3(kRowThreads), 0, st, a); \
    }
    FLK_NORM_PLANS(FLK_CALL)
#undef FLK_CALL
}
template <typename T, int VEC> void norm_backward(const NormArgs<T> &a, const NormPlan &plan, int64_t groups, hipStream_t st) {
#define FLK_CALL(TPR, NV)                                                                                              \
    if constexpr (NV == 0) {                                                                                           \
        if (a.rows > 0)                                                                                                \
            hipLaunchKernelGGL((layer_norm_bwd_long_kernel<T>), dim3((unsigned)norm_min(a.rows, 4096)), dim3(kLoopThreads), 0, st, a); \
        if (a.partial != nullptr)                                                                                      \
            hipLaunchKernelGGL((layer_norm_columns_kernel<T>), dim3((unsigned)((a.d + kRowThreads - 1) / kRowThreads), (unsigned)groups), \
                               dim3(kRowThreads), 0, st, a);                                                           \
    } else {                                                                                                           \
        hipLaunchKernelGGL((layer_norm_bwd_kernel<T, VEC, TPR, NV>), dim3((unsigned)groups), dim3(kRowThreads), 0, st, a); \
    }
    FLK_NORM_PLANS(FLK_CALL)
#undef FLK_CALL
}

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
constexpr int64_t kNormMaxD = (int64_t)1 << 30;

template <typename T>
static bool norm_aligned(int64_t d, const void *x, int64_t x_rs, const void *dy, int64_t dy_rs, const void *y, const void *w,
                         const void *b) {
    constexpr int vec = 16 / sizeof(T);
    return d % vec == 0 && x_rs % vec == 0 && dy_rs % vec == 0 && aligned16(x) && aligned16(dy) && aligned16(y) && aligned16(w) &&
           aligned16(b);
}

template <typename T>
static int norm_fwd_impl(const void *x, int64_t rows, int64_t d, int64_t x_rs, const void *w, const void *b, int wide, double eps,
                         void *y, void *mean, void *rstd, hipStream_t st) {
    const NormPlan plan = norm_plan<T>(d, norm_aligned<T>(d, x, x_rs, nullptr, 0, y, w, b));
    typedef typename NormAcc<T>::type A;
    NormArgs<T> a{(const T *)x, nullptr, (T *)y, w, b, (A *)mean, (A *)rstd, nullptr, nullptr, rows, d, x_rs, 0, wide, eps};
    if (plan.vec == 1) norm_forward<T, 1>(a, plan, st);
    else norm_forward<T, 16 / sizeof(T)>(a, plan, st);
    FLK_LAUNCH_CHECK("layer_norm_kernel");
    return FLK_OK;
}

template <typename T>
static size_t norm_bwd_bytes(int64_t rows, int64_t d) {        // enough for either row layout
    const NormPlan plan = norm_plan<T>(d, false);
    const int64_t n = norm_bwd_groups(rows, norm_plan<T>(d, true)), m = norm_bwd_groups(rows, plan);
    return ((size_t)(n > m ? n : m) * 2 * (size_t)d + (size_t)(plan.nv == 0 ? rows : 0)) * sizeof(typename NormAcc<T>::type);
}

template <typename T>
static int norm_bwd_impl(const void *x, int64_t rows, int64_t d, int64_t x_rs, const void *dy, int64_t dy_rs, const void *w,
                         int wide, const void *mean, const void *rstd, void *dx, void *dw, void *db, void *ws, size_t ws_bytes,
                         hipStream_t st) {
    typedef typename NormAcc<T>::type A;
    const bool sums = dw != nullptr || db != nullptr;
    if (sums && (ws == nullptr || ws_bytes < norm_bwd_bytes<T>(rows, d)))
        return fail(FLK_ENOMEM, "workspace of %zu bytes given, %zu needed", ws_bytes, norm_bwd_bytes<T>(rows, d));
    const NormPlan plan = norm_plan<T>(d, norm_aligned<T>(d, x, x_rs, dy, dy_rs, dx, w, nullptr));
    const int64_t groups = norm_bwd_groups(rows, plan);
    NormArgs<T> a{(const T *)x, (const T *)dy, (T *)dx, w, nullptr, (A *)mean, (A *)rstd, sums ? (A *)ws : nullptr, nullptr, rows, d,
                  x_rs, dy_rs, wide, 0.0};
    if (sums && plan.nv == 0) a.shift = a.partial + groups * 2 * d;
    if (plan.vec == 1) norm_backward<T, 1>(a, plan, groups, st);
    else norm_backward<T, 16 / sizeof(T)>(a, plan, groups, st);
    FLK_LAUNCH_CHECK("layer_norm_bwd_kernel");
    if (!sums) return FLK_OK;
    const dim3 grid((unsigned)((2 * d + 31) / 32));
    if (wide || sizeof(T) == 4) {
        hipLaunchKernelGGL((layer_norm_finish_kernel<T, float>), grid, dim3(1024), 0, st, (const A *)ws, (int)groups, d, (float *)dw, (float *)db);
    } else {
        hipLaunchKernelGGL((layer_norm_finish_kernel<T, T>), grid, dim3(1024), 0, st, (const A *)ws, (int)groups, d, (T *)dw, (T *)db);
    }
    FLK_LAUNCH_CHECK("layer_norm_finish_kernel");
    return FLK_OK;
}

static int norm_check(const char *what, int64_t rows, int64_t d, int64_t rs, int dtype, int w_dtype, const void *w, const void *b) {
    if (rows < 0) return fail(FLK_EINVAL, "%s: negative number of rows", what);
    if (d < 1) return fail(FLK_EINVAL, "%s: feature dimension must be positive", what);
    if (d > kNormMaxD) return fail(FLK_EUNSUPPORTED, "%s: more than %lld features", what, (long long)kNormMaxD);
    if (rs < 0) return fail(FLK_EINVAL, "%s: negative row stride", what);
    if (dtype != FLK_F32 && dtype != FLK_F64 && dtype != FLK_F16 && dtype != FLK_BF16)
        return fail(FLK_EINVAL, "unknown dtype %d", dtype);
    if ((w != nullptr || b != nullptr) && w_dtype != dtype && !(w_dtype == FLK_F32 && dtype != FLK_F64))
        return fail(FLK_EINVAL, "%s: the weight is of the data's type or, for 16-bit data, float", what);
    return FLK_OK;
}

}  // namespace flk

using namespace flk;

extern "C" {

int flk_layer_norm(const void *x, int64_t rows, int64_t d, int64_t x_rs, const void *weight, const void *bias, int weight_dtype,
                   double eps, void *y, void *mean, void *rstd, int dtype, void *stream) {
    fail(FLK_OK, "%s", "");
    const int rc = norm_check("flk_layer_norm", rows, d, x_rs, dtype, weight_dtype, weight, bias);
    if (rc != FLK_OK || rows == 0) return rc;
    if (!(eps >= 0.0)) return fail(FLK_EINVAL, "flk_layer_norm: eps must not be negative");
    if (x == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr)) return fail(FLK_EINVAL, "flk_layer_norm: null pointer");
    hipStream_t st = (hipStream_t)stream;
    const int wide = weight_dtype == FLK_F32 && dtype != FLK_F32;
    if (dtype == FLK_F32) return norm_fwd_impl<float>(x, rows, d, x_rs, weight, bias, wide, eps, y, mean, rstd, st);
    if (dtype == FLK_F64) return norm_fwd_impl<double>(x, rows, d, x_rs, weight, bias, 0, eps, y, mean, rstd, st);
    if (dtype == FLK_F16) return norm_fwd_impl<f16_t>(x, rows, d, x_rs, weight, bias, wide, eps, y, mean, rstd, st);
    return norm_fwd_impl<bf16_t>(x, rows, d, x_rs, weight, bias, wide, eps, y, mean, rstd, st);
}

size_t flk_layer_norm_backward_workspace_bytes(int64_t rows, int64_t d, int dtype) {
    if (rows < 0 || d < 1 || d > kNormMaxD) return 0;
    if (dtype == FLK_F32) return norm_bwd_bytes<float>(rows, d);
    if (dtype == FLK_F64) return norm_bwd_bytes<double>(rows, d);
    if (dtype == FLK_F16 || dtype == FLK_BF16) return norm_bwd_bytes<f16_t>(rows, d);
    return 0;
}

int flk_layer_norm_backward(const void *x, int64_t rows, int64_t d, int64_t x_rs, const void *dy, int64_t dy_rs, const void *weight,
                            int weight_dtype, const void *mean, const void *rstd, void *dx, void *dweight, void *dbias, int dtype,
                            void *workspace, size_t workspace_bytes, void *stream) {
    fail(FLK_OK, "%s", "");
    const int rc = norm_check("flk_layer_norm_backward", rows, d, x_rs, dtype, weight_dtype, weight, dweight != nullptr ? dweight : dbias);
    if (rc != FLK_OK) return rc;
    if (dy_rs < 0) return fail(FLK_EINVAL, "flk_layer_norm_backward: negative row stride");
    if (rows > 0 && (x == nullptr || dy == nullptr || mean == nullptr || rstd == nullptr))
        return fail(FLK_EINVAL, "flk_layer_norm_backward: null pointer");
    if (dx == nullptr && dweight == nullptr && dbias == nullptr) return FLK_OK;
    hipStream_t st = (hipStream_t)stream;
    const int wide = weight_dtype == FLK_F32 && dtype != FLK_F32;
#define FLK_CALL(T, W) norm_bwd_impl<T>(x, rows, d, x_rs, dy, dy_rs, weight, W, mean, rstd, dx, dweight, dbias, workspace, workspace_bytes, st)
    if (dtype == FLK_F32) return FLK_CALL(float, wide);
    if (dtype == FLK_F64) return FLK_CALL(double, 0);
    if (dtype == FLK_F16) return FLK_CALL(f16_t, wide);
    return FLK_CALL(bf16_t, wide);
#undef FLK_CALL
}

}  // extern "C"
