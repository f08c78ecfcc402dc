// Tiles, matrix-core fragments, masks and scores shared by the attention kernels (gfx950).
//
//   x_ij  = scale * q_i.k_j;   x <- cap * tanh(x / cap)  (cap > 0);   x <- x - slope_h * |pos_i - j|  (slopes given)
//   out_i = sum_j p_ij v_j,    p_ij = exp(x_ij - lse_i) over the keys j that row i sees
//   row i stands at pos_i = i + (sk - sq): the queries are the newest of the sk positions.
//
// All products run on 32x32 matrix instructions in the orientation that leaves the softmax rows on lanes: the scores are
// formed transposed, S^T = K Q^T, so that lane (l & 31) holds one query and its registers the keys.  A row's maximum and sum are
// then register operations plus one exchange between the two lane halves, and the accumulator registers are, packed, the
// second operand of the next product (O^T = V^T P^T) without any movement between lanes: register r of half h is key
// 8 (r / 4) + 4 h + r % 4, and the order of the terms of a product does not matter as long as both operands use the same.
#pragma once
#include "flk_common.h"
#include "element_types.h"

namespace flk {

typedef float fx16 __attribute__((ext_vector_type(16)));
typedef float fx4 __attribute__((ext_vector_type(4)));
typedef f16_t hx8 __attribute__((ext_vector_type(8)));
typedef bf16_t bx8 __attribute__((ext_vector_type(8)));
typedef short sx4 __attribute__((ext_vector_type(4)));
typedef unsigned ux4 __attribute__((ext_vector_type(4)));

constexpr float kScoreUnit = 1.44269504088896340736f;   // log2(e): scores are kept in units of log 2
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff();
constexpr int kAttnThreads = 256;          // four waves of 32 rows (queries, or keys in the dk / dv kernel)
constexpr int kAttnRows = 128;
constexpr int kAttnMaxD = 128;
constexpr int kDocBlock = 32;              // positions one entry of the document ranges covers

// A fragment is 16 bytes of a row: lane half h holds KS / 2 consecutive values of a KS-wide step.
template <typename T> struct AttnType;
template <> struct AttnType<float> {
    typedef fx4 frag;
    static constexpr int E = 4, KS = 8, kTile = 32;
    static __device__ __forceinline__ fx16 mma(frag a, frag b, fx16 c) {
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ bool finite(float x) { return __builtin_isfinite(x); }
};
template <> struct AttnType<f16_t> {
    typedef hx8 frag;
    static constexpr int E = 8, KS = 16, kTile = 64;
    static __device__ __forceinline__ fx16 mma(frag a, frag b, fx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct AttnType<bf16_t> {
    typedef bx8 frag;
    static constexpr int E = 8, KS = 16, kTile = 64;
    static __device__ __forceinline__ fx16 mma(frag a, frag b, fx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// Whether any value of 16 bytes is an infinity or a NaN: its exponent bits are all ones.
template <typename T> __device__ __forceinline__ bool any_nonfinite(ux4 u) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) bad |= (u[i] & 0x7f800000u) == 0x7f800000u;
        else {
            constexpr unsigned m = std::is_same<T, f16_t>::value ? 0x7c00u : 0x7f80u;
            bad |= (u[i] & m) == m || (u[i] >> 16 & m) == m;
        }
    }
    return bad;
}

// A tile of rows in LDS, `DP` values each.  Its 16-byte chunks are permuted within a row by an exclusive or with swz(row):
// eight consecutive rows put the same chunk into different banks (row-wise fragments), and four consecutive rows put
// the same pair of chunks into different banks (fragments read across the rows).
template <typename T, int DP> struct Tile {
    static constexpr int RB = DP * (int)sizeof(T), NC = RB / 16;
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (RB % 128 == 0) return (r & 3) << 1 | (r >> 2 & 1);
        else return (r & 2) | (r >> 2 & 1);        // rows of 64 or 192 bytes already alternate between two halves of the banks
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swz(row)) << 4); }

    typedef typename AttnType<T>::frag frag;
    // step c of the row of this lane (row0 + lane % 32)
    static __device__ __forceinline__ frag rows(const char *tile, int row0, int c) {
        const int l = threadIdx.x & 63;
        return *(const frag *)(tile + at(row0 + (l & 31), 2 * c + (l >> 5)));
    }
    // columns d0 + lane % 32 of KS rows from row0 on, in the order in which the accumulator registers hold rows
    static __device__ __forceinline__ frag cols(const char *tile, int row0, int d0) {
        const int l = threadIdx.x & 63, h = l >> 5;
        frag f;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int c = d0 + (l & 31);
                f[i] = *(const float *)(tile + at(row0 + 4 * h + i, c >> 2) + (c & 3) * 4);
            }
        } else {
            // the transposing read: of 16 lanes, four each name 4 values of one row; lane i gets column i of the four rows
            const int i = l & 15, b = (d0 + (l & 16)) * 2 + (i & 3) * 8;
            union { sx4 s[2]; frag f; } u;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const char *p = tile + at(row0 + 8 * k + 4 * h + (i >> 2), b >> 4) + (b & 8);
                u.s[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sx4 *)p);
            }
            f = u.f;
        }
        return f;
    }
};

// KS accumulator registers from r0 on as the second operand of a product over their rows.  The rounding of p (and of its
// gradient) to 16 bits is what feeds the matrix cores at their full rate; p lies in [0, 1] before the final division, its
// rounding errors are independent, and the sums of p itself are of the unrounded values.
template <typename T> __device__ __forceinline__ typename AttnType<T>::frag pack(const fx16 &x, int s) {
    typename AttnType<T>::frag f;
    constexpr int n = AttnType<T>::E;
#pragma unroll
    for (int i = 0; i < n; i++) f[i] = (T)x[n * s + i];
    return f;
}

// Product with rows that may hold infinities or NaNs in places this step's weights hide: those get no share, and where a
// weight that is not zero meets one, the sum becomes what the formula gives.
template <typename T>
__device__ __forceinline__ fx16 mma_careful(typename AttnType<T>::frag a, typename AttnType<T>::frag p, fx16 c) {
    typename AttnType<T>::frag up = a, down = a, seen = p;
#pragma unroll
    for (int i = 0; i < AttnType<T>::E; i++) {
        const float x = (float)a[i];
        const bool fine = __builtin_fabsf(x) < kInf;
        up[i] = (T)(fine || x == -kInf ? 0.f : 1.f);
        down[i] = (T)(fine || x == kInf ? 0.f : 1.f);
        seen[i] = (T)((float)p[i] == 0.f ? 0.f : 1.f);
        if (!fine) a[i] = (T)0.f;
    }
    fx16 u = {}, d = {};
    c = AttnType<T>::mma(a, p, c);
    u = AttnType<T>::mma(up, seen, u);
    d = AttnType<T>::mma(down, seen, d);
#pragma unroll
    for (int i = 0; i < 16; i++) {
        if (u[i] > 0.f) c[i] += kInf;
        if (d[i] > 0.f) c[i] -= kInf;
    }
    return c;
}

struct AttnStride { int64_t b, s, h; };
struct AttnArgs {
    const void *q, *k, *v, *out, *dout;
    void *o, *dq, *dk, *dv;
    float *lse, *delta, *dslopes_part, *dkv_part;
    AttnStride qs, ks, vs, os, dos;                    // strides of q, k, v, out and dout; the gradients are contiguous
    int b, sq, sk, hq, hk, group, d, dv_d;
    int splits;                                        // dk / dv: parts the heads of a group are divided into
    float scale, cap;
    const float *slopes;
    const int *prefix, *docs;
    int64_t docs_b;
    int2 *doc_range;                                   // [b][blocks of kDocBlock positions]
    int doc_blocks;
    int causal, vec;                                   // vec: all rows can be read 16 bytes at a time
};

// 16 bytes of a row from value c * E on; zero past the row's end.  Rows that are not aligned are read value by value.
template <typename T> __device__ __forceinline__ ux4 load_chunk(const T *row, int c, int d, bool live, int vec) {
    constexpr int E = AttnType<T>::E;
    ux4 r = {0, 0, 0, 0};
    if (live && c * E < d) {
        if (vec) r = *(const ux4 *)(row + c * E);
        else {
            union { T t[E]; ux4 u; } x;
            x.u = r;
#pragma unroll
            for (int i = 0; i < E; i++)
                if (c * E + i < d) x.t[i] = row[c * E + i];
            r = x.u;
        }
    }
    return r;
}

// The share of this thread in a tile of TR rows: global memory to registers, later registers to LDS.
template <typename T, int DP, int TR> struct Stage {
    static constexpr int NC = Tile<T, DP>::NC, N = (TR * NC + kAttnThreads - 1) / kAttnThreads;
    ux4 r[N];
    __device__ __forceinline__ void load(const T *base, int64_t stride, int rows, int d, int vec) {
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int i = n * kAttnThreads + threadIdx.x, row = i / NC, c = i % NC;
            r[n] = load_chunk<T>(base + row * stride, c, d, row < rows && i < TR * NC, vec);
        }
    }
    __device__ __forceinline__ void store(char *tile) const {
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int i = n * kAttnThreads + threadIdx.x, row = i / NC, c = i % NC;
            if (TR * NC % kAttnThreads == 0 || i < TR * NC) *(ux4 *)(tile + Tile<T, DP>::at(row, c)) = r[n];
        }
    }
    __device__ __forceinline__ bool nonfinite() const {
        bool bad = false;
#pragma unroll
        for (int n = 0; n < N; n++) bad |= any_nonfinite<T>(r[n]);
        return bad;
    }
};

// tanh through one exponential; near zero, where 1 - 2 / (1 + e) would cancel, the odd series (next term below 2^-25 at 1/4)
template <typename T> __device__ __forceinline__ float tanh_of(float u) {
    const float e = __builtin_amdgcn_exp2f(2.f * kScoreUnit * u);
    const float t = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e);
    if constexpr (sizeof(T) == 2) return t;
    const float w = u * u;
    const float s = u * (1.f + w * (-1.f / 3 + w * (2.f / 15 + w * (-17.f / 315 + w * (62.f / 2835)))));
    return __builtin_fabsf(u) < 0.25f ? s : t;
}

// One score in units of log 2, and the tanh (for its derivative)
template <typename T, bool MOD>
__device__ __forceinline__ float score(const AttnArgs &p, float s, float slope, int pos, int key, float &t) {
    if constexpr (!MOD) return s * (p.scale * kScoreUnit);
    float x = s * p.scale;
    if (p.cap > 0.f) { t = tanh_of<T>(x * __builtin_amdgcn_rcpf(p.cap)); x = p.cap * t; }
    return (x - slope * __builtin_fabsf((float)(pos - key))) * kScoreUnit;
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o, 64));
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = max(x, __shfl_xor(x, o, 64));
    return __builtin_amdgcn_readfirstlane(x);
}

// smallest and largest document id of positions [lo, hi), a padding position counting as -1; (0, -1) if there is none
__device__ __forceinline__ int2 doc_span(const int2 *range, int lo, int hi) {
    int2 s = {0x7fffffff, -1};
    for (int b = lo / kDocBlock; b * kDocBlock < hi; b++) { s.x = min(s.x, range[b].x); s.y = max(s.y, range[b].y); }
    return s;
}
__device__ __forceinline__ bool docs_meet(int2 a, int2 b) { return a.y >= 0 && b.y >= 0 && a.x <= b.y && b.x <= a.y; }

constexpr int kCachedKeys = 32;            // keys of a wave's tile

struct CachedArgs {
    const void *q, *k, *v;
    void *out;
    AttnStride qs, ks, vs;                 // q: [b][t][hq][d]
    const int *lengths;
    const float *slopes;
    float *part_o, *part_ml;               // parts of several workgroups: [row][split][dv] and [row][split][2]
    int b, t, capacity, hq, hk, group, d, dv_d, splits, blocks_r;
    float scale, cap;
    int vec;
};

// What the kernels look like from a launcher (attention.hip); one source per element type instantiates them.
template <typename T> int launch_attention_fwd(const AttnArgs &a, int dp, hipStream_t st);
template <typename T> int launch_attention_dq(const AttnArgs &a, int dp, hipStream_t st);
template <typename T> int launch_attention_dkv(const AttnArgs &a, int dp, hipStream_t st);
template <typename T> int launch_attention_cached(const CachedArgs &a, int dp, hipStream_t st);

#define FLK_ATTN_LAUNCH(KERNEL, GRID)                                                                                        \
    const bool mod = a.cap > 0.f || a.slopes != nullptr;                                                                     \
    if (dp == 32) { if (mod) hipLaunchKernelGGL((KERNEL<T, 32, true>), GRID, dim3(kAttnThreads), 0, st, a);                  \
                    else hipLaunchKernelGGL((KERNEL<T, 32, false>), GRID, dim3(kAttnThreads), 0, st, a); }                   \
    else if (dp == 64) { if (mod) hipLaunchKernelGGL((KERNEL<T, 64, true>), GRID, dim3(kAttnThreads), 0, st, a);             \
                         else hipLaunchKernelGGL((KERNEL<T, 64, false>), GRID, dim3(kAttnThreads), 0, st, a); }              \
    else if (dp == 96) { if (mod) hipLaunchKernelGGL((KERNEL<T, 96, true>), GRID, dim3(kAttnThreads), 0, st, a);             \
                         else hipLaunchKernelGGL((KERNEL<T, 96, false>), GRID, dim3(kAttnThreads), 0, st, a); }              \
    else { if (mod) hipLaunchKernelGGL((KERNEL<T, 128, true>), GRID, dim3(kAttnThreads), 0, st, a);                          \
           else hipLaunchKernelGGL((KERNEL<T, 128, false>), GRID, dim3(kAttnThreads), 0, st, a); }                           \
    FLK_LAUNCH_CHECK(#KERNEL);                                                                                               \
    return FLK_OK;

#if defined(FLK_KF)
#if FLK_KF == 0
typedef float attn_t;
#elif FLK_KF == 1
typedef f16_t attn_t;
#else
typedef bf16_t attn_t;
#endif
#endif

}  // namespace flk
