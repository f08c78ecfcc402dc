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
typedef ux4 ux4_any2 __attribute__((aligned(2)));          // at any address of a 2 (4) byte value
typedef ux4 ux4_any4 __attribute__((aligned(4)));

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
    typedef ux4_any4 any;
    static constexpr int E = 4, KS = 8, kTile = 32, M = 4, R = 4;   // M, R: matrix instructions and cross-row reads a fragment
    static __device__ __forceinline__ fx16 mma(frag a, frag b, fx16 c) {
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ bool finite(float x) { return __builtin_isfinite(x); }
};
template <> struct AttnType<f16_t> {
    typedef hx8 frag;
    typedef ux4_any2 any;
    static constexpr int E = 8, KS = 16, kTile = 64, M = 1, R = 2;
    static __device__ __forceinline__ fx16 mma(frag a, frag b, fx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct AttnType<bf16_t> {
    typedef bx8 frag;
    typedef ux4_any2 any;
    static constexpr int E = 8, KS = 16, kTile = 64, M = 1, R = 2;
    static __device__ __forceinline__ fx16 mma(frag a, frag b, fx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// Whether values are infinities or NaNs: their exponent bits are all ones, and one more in the last of them carries into the
// sign's place.  Gathered over many chunks by bad_bits, asked once by any_bad.
template <typename T> __device__ __forceinline__ unsigned bad_bits(ux4 u) {
    constexpr unsigned m = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, f16_t>::value ? 0x7c007c00u : 0x7f807f80u;
    constexpr unsigned one = m & (0u - m), step = sizeof(T) == 4 ? one : one | one << 16;
    unsigned r = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) r |= (u[i] & m) + step;
    return r;
}
template <typename T> __device__ __forceinline__ bool any_bad(unsigned bits) { return (bits & (sizeof(T) == 4 ? 0x80000000u : 0x80008000u)) != 0; }
template <typename T> __device__ __forceinline__ bool any_nonfinite(ux4 u) { return any_bad<T>(bad_bits<T>(u)); }

// A tile of rows in LDS, `DP` values each.  Its 16-byte chunks are permuted within a row by an exclusive or with swz(row), so that
// what is read in one cycle, 256 bytes from all 64 banks, lies in different banks: one chunk of 16 rows (row-wise fragments)
// and four neighbouring chunks of four rows (fragments read across the rows).  Rows of less than 256 bytes begin in
// different banks already and need fewer bits.  (128 16-bit values a row: 4 and 2 cycles a fragment's instruction where eight
// permuted rows gave 8 and 4.)  For float, whose matrix instructions take 16 times as long, eight rows are enough.
template <typename T, int DP> struct Tile {
    static constexpr int RB = DP * (int)sizeof(T), NC = RB / 16;
    static constexpr int XB = sizeof(T) == 4 ? 3 : RB % 256 == 0 ? 4 : RB % 128 == 0 ? 3 : 2;      // chunk bits that are permuted
    static constexpr int kPeriod = sizeof(T) == 4 ? 8 : 16;                                        // rows after which it repeats
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (sizeof(T) == 4) return (r & 3) << 1 | (r >> 2 & 1);
        else if constexpr (XB == 4) return (r & 3) << 2 | (r >> 2 & 3);
        else if constexpr (XB == 3) return (r >> 1 & 1) << 2 | (r >> 2 & 3);
        else return r >> 2 & 3;
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swz(row)) << 4); }

    typedef typename AttnType<T>::frag frag;
    // This lane's places in a tile: of chunk `half` of its row, and of its part of a fragment across the first rows.  The bits
    // that are permuted lie below a row's, so an exclusive or with a constant leads to every other fragment.
    static constexpr int RV = 1 << (XB - 1), DV = 1 << (XB - 2);
    struct Lane {
        int r, c;
        __device__ __forceinline__ void init() {
            const int l = threadIdx.x & 63, h = l >> 5, m = l & 31;
            r = at(m, h);
            if constexpr (sizeof(T) == 4) c = at(4 * h, m >> 2) + (m & 3) * 4;
            // the transposing read: of 16 lanes, four each name 4 values of one row; lane i gets column i of the four rows
            else c = at(4 * h + (l >> 2 & 3), 2 * (l >> 4 & 1) + (l >> 1 & 1)) + (l & 1) * 8;
        }
        // keeps the compiler from holding all the derived places in registers for the whole of a loop
        __device__ __forceinline__ void renew() { asm volatile("" : "+v"(r), "+v"(c)); }
    };
    // step c of the row of this lane (row0 + lane % 32; row0 a multiple of 32)
    static __device__ __forceinline__ frag rows(const char *tile, const Lane &p, int row0, int c) {
        return *(const frag *)(tile + (p.r ^ (c % RV * 32)) + row0 * RB + c / RV * RV * 32);
    }
    // columns 32 db + lane % 32 of KS rows from row0 on (a multiple of KS), in the order in which the accumulator registers
    // hold rows
    static __device__ __forceinline__ frag cols(const char *tile, const Lane &p, int row0, int db) {
        frag f;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) f[i] = *(const float *)(tile + (p.c ^ (i * 32)) + (row0 + i) * RB + db * 128);
        } else {
            union { sx4 s[2]; frag f; } u;
#pragma unroll
            for (int k = 0; k < 2; k++)
                u.s[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sx4 *)(
                    tile + (p.c ^ (db % DV * 64 + k * 32)) + (row0 + 8 * k) * RB + db / DV * DV * 64));
            f = u.f;
        }
        return f;
    }
};

// Whether the type's range is narrow: float16's normal numbers end at 6e-5, which the weights of a row of 16 000 keys reach, and rounding
// below that costs digits (below 3e-8, everything).  Its weights are held times 2^8 or more where they are rounded; the shift is a part of
// the exponent and costs nothing.
template <typename T> constexpr bool kNarrow = std::is_same<T, f16_t>::value;

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

// Infinities and NaNs of a tile must not reach rows that hide them, but a product with weight zero would carry them there.
// They are set to zero where a mask is needed; cleaned() does it to 16 bytes, clean() to this thread's 16 bytes of LDS.
template <typename T> __device__ __forceinline__ ux4 cleaned(ux4 u) {
    union { ux4 u; T t[16 / sizeof(T)]; } x;
    x.u = u;
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); i++)
        if (!(__builtin_fabsf((float)x.t[i]) < kInf)) x.t[i] = (T)0.f;
    return x.u;
}
template <typename T> __device__ __forceinline__ void clean(char *at) {
    const ux4 u = *(const ux4 *)at;
    if (any_nonfinite<T>(u)) *(ux4 *)at = cleaned<T>(u);
}

struct AttnStride { int64_t b, s, h; };
struct AttnArgs {
    const void *q, *k, *v, *out, *dout;
    void *o, *rest, *dq, *dk, *dv;                     // rest: what rounding took from out, for the backward pass
    float *lse, *dslopes_part, *dq_part, *dkv_part;
    // backward: [b][hq][3][sq_pad], the rows' lse (in units of log 2; infinite, so that weights are zero, for a row of q or dout that holds
    // infinities or NaNs), delta, and the lse without that
    float *stats;
    float2 *sizes;                                     // backward of float16: [b][hq][sq_pad / 32], largest norm of 32 rows of dout (negative: bad_rows) and |delta|
    unsigned char *bad_rows;                           // backward: [b][hq][sq_pad / 32], whether there is such a row among 32 (1) that sees something (2)
    int64_t sq_pad;
    AttnStride qs, ks, vs, dos;                        // strides of q, k, v and dout; the others are contiguous
    int b, sq, sk, hq, hk, group, d, dv_d;
    // Workgroups that share a tile's rows, each with a part of its tiles of keys (forward, dq): parts; dk / dv: head_parts, each with
    // a part of the heads of the group, times row_parts, each with a part of the tiles of queries
    int parts, head_parts, row_parts;
    float *part_o, *part_ml;                           // forward: [part][b][sq][hq][dv] and [part][b][sq][hq][2], maximum and sum
    float scale, cap;
    const float *slopes;
    const int *prefix, *docs;
    int64_t docs_b;
    int2 *doc_range;                                   // [b][doc_blocks]: smallest and largest id of kDocBlock positions
    int *doc_ids;                                      // [b][doc_blocks * kDocBlock]: the ids, -1 for padding and past the end
    int doc_blocks;
    int causal;
    int vec, vec_v;                                    // rows of q and k (of v and what is like it) are whole aligned chunks
};

// 16 bytes of a row from value c * E on; zero past the row's end.  The hardware reads them from any address; where a row does not
// end with a chunk (vec: it does), its last values are read one by one.
template <typename T> __device__ __forceinline__ ux4 load_chunk(const T *row, int c, int d, bool live, int vec) {
    constexpr int E = AttnType<T>::E;
    ux4 r = {0, 0, 0, 0};
    if (live && c * E < d) {
        if (vec) r = *(const ux4 *)(row + c * E);
        else if (c * E + E <= d) r = *(const typename AttnType<T>::any *)(row + c * E);
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

// Tiles of TR rows on their way into LDS.  Aligned rows go there directly, 16 bytes a lane, without passing through registers:
// a wave's instruction fills 1024 consecutive bytes of LDS, so the permutation of the chunks is applied to the addresses
// read.  Lanes past the last row or the row's end read out of the buffer's bounds and bring zeros.  The reads are counted by
// vmcnt; wait() and a barrier stand between them and the tile's use.  Their targets are named by 16 bits, so tiles lie in the first
// 64 KB of LDS.  Other rows pass through registers.
constexpr unsigned kNowhere = 0x80000000u;                 // an offset behind every buffer's end
template <typename T, int DP, int TR> struct Feed {
    typedef Tile<T, DP> TL;
    static constexpr int NC = TL::NC, N = TR * NC / kAttnThreads, kStep = kAttnThreads / NC;
    static_assert(TR * NC % kAttnThreads == 0, "every instruction is full");
    static constexpr bool kEven = kAttnThreads % NC == 0 && kStep % TL::kPeriod == 0;   // all instructions permute alike
    const T *base;
    int64_t stride;
    unsigned off[kEven ? 1 : N];
    int d, vec;
    __device__ __forceinline__ void init(const T *b, int64_t st, int d_, int vec_) {
        base = b; stride = st; d = d_; vec = vec_;
#pragma unroll
        for (int n = 0; n < (kEven ? 1 : N); n++) {
            const int i = n * kAttnThreads + threadIdx.x, row = i / NC, c = i % NC ^ TL::swz(row);
            off[n] = c * AttnType<T>::E < d ? (unsigned)(row * (int)(stride * sizeof(T)) + c * 16) : kNowhere;
        }
    }
    __device__ __forceinline__ void issue(char *tile, int row0, int rows) const {
        if (vec) {
            const uint64_t a = (uint64_t)(base + row0 * stride);
            ux4 rsrc;
            rsrc[0] = __builtin_amdgcn_readfirstlane((unsigned)a);
            rsrc[1] = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32) & 0xffffu);
            rsrc[2] = 0x7fffffffu;
            rsrc[3] = 0x00027000u;
            const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)tile +
                                                               (threadIdx.x & ~63u) * 16);
            const int step = __builtin_amdgcn_readfirstlane((int)(kStep * stride * sizeof(T)));
#pragma unroll
            for (int n = 0; n < N; n++) {
                unsigned o = off[kEven ? 0 : n];
                if (rows < TR && (n * kAttnThreads + (int)threadIdx.x) / NC >= rows) o = kNowhere;
                const int so = kEven ? n * step : 0;
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                             :: "s"(to + n * kAttnThreads * 16), "v"(o), "s"(rsrc), "s"(so) : "memory", "m0");
            }
        } else {
            constexpr int B = N % 4 == 0 ? 4 : N % 3 == 0 ? 3 : N % 2 == 0 ? 2 : 1;      // reads on their way at once
#pragma unroll 1
            for (int n0 = 0; n0 < N; n0 += B) {
                ux4 t[B];
#pragma unroll
                for (int n = 0; n < B; n++) {
                    const int i = (n0 + n) * kAttnThreads + threadIdx.x, row = i / NC, c = i % NC;
                    t[n] = load_chunk<T>(base + (row0 + row) * stride, c, d, row < rows, 0);
                }
#pragma unroll
                for (int n = 0; n < B; n++) {
                    const int i = (n0 + n) * kAttnThreads + threadIdx.x;
                    *(ux4 *)(tile + TL::at(i / NC, i % NC)) = t[n];
                }
            }
        }
    }
    // (the builtin, which the compiler counts: it would wait again for whatever it takes to be still on its way)
    static __device__ __forceinline__ void wait() { __builtin_amdgcn_s_waitcnt(0x0f70); asm volatile("" ::: "memory"); }
    static __device__ __forceinline__ void clean_share(char *tile) {
#pragma unroll
        for (int n = 0; n < N; n++) clean<T>(tile + (n * kAttnThreads + threadIdx.x) * 16);
    }
    // 32 rows of a tile (the rows of a block of products), by all of the workgroup's threads, once they have been read as they came
    static __device__ __forceinline__ void clean_block(char *tile, int block) {
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * NC; i += kAttnThreads) clean<T>(tile + (block * 32 * NC + i) * 16);
        __syncthreads();
    }
    // whether this thread's share of a tile in LDS holds an infinity or a NaN
    static __device__ __forceinline__ bool nonfinite(const char *tile) {
        unsigned bits = 0;
#pragma unroll
        for (int n = 0; n < N; n++) bits |= bad_bits<T>(*(const ux4 *)(tile + (n * kAttnThreads + threadIdx.x) * 16));
        return any_bad<T>(bits);
    }
};

// A wave's 32 rows of results, which lie in registers four values at a time (value 32 db + 8 g + 4 half + i of row lane % 32 in
// x[db][4 g + i]), to memory in whole rows: through 32 rows of a tile in LDS that belong to this wave alone.  Written from the
// registers, a row of 128 16-bit values would be 64 stores of two bytes (2048 workgroups: 80 us for nothing but that).
// part(db, r): the value to write.
template <typename T, int DP, typename Part>
__device__ __forceinline__ void store_rows(char *lds, Part part, T *out, int64_t stride, int rows, int d, int vec) {
    typedef Tile<T, DP> TL;
    constexpr int E = AttnType<T>::E, NC = TL::NC;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");         // what was read there before has been read
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int db = 0; db < DP / 32; db++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int c = 32 * db + 8 * g + 4 * half;
            struct alignas(4 * sizeof(T)) { T t[4]; } x;
#pragma unroll
            for (int i = 0; i < 4; i++) x.t[i] = (T)part(db, 4 * g + i);
            *(decltype(x) *)(lds + TL::at(lane & 31, c / E) + c % E * (int)sizeof(T)) = x;
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll 4
    for (int i = lane; i < 32 * NC; i += 64) {
        const int row = i / NC, c = i % NC;
        if (row >= rows || c * E >= d) continue;
        const char *from = lds + TL::at(row, c);
        T *to = out + row * stride + c * E;
        if (vec) *(ux4 *)to = *(const ux4 *)from;
        else if (c * E + E <= d) *(typename AttnType<T>::any *)to = *(const ux4 *)from;
        else
            for (int j = 0; j < E && c * E + j < d; j++) to[j] = ((const T *)from)[j];
    }
}

// What happens to the scores before the softmax.  A scale that is not positive goes with kDecay, whose rows look for their
// maximum among the finished scores.
constexpr int kPlain = 0, kCap = 1, kDecay = 2, kCapDecay = 3;

// Scores x in units of log 2, and the derivative of the cap.  With r = 1 / (1 + exp(2 u)), u = scale s / cap:
// cap tanh u = cap - 2 cap r, and its derivative in u is 4 cap r (1 - r).  Two transcendental instructions a score; r comes with an
// error of 2^-24, so a score with one of cap 2^-22, far below what rounding the weights to 16 bits costs for caps up to
// kMaxCap16.  Float data take the odd
// series instead where tanh is small and 1 - 2 r would cancel (its next term is below 2^-25 of the sum at u = 1/4).
// Within kMaxScale and the caps' limits, 2 log2(e) scale / cap and log2(e) cap are numbers of float.
constexpr double kMaxCap16 = 4096.0, kMinCap = 1e-20, kMaxCap = 1e20, kMaxScale = 1e18;
template <typename T, int MOD> struct Score {
    static constexpr bool kHasCap = (MOD & 1) != 0, kHasDecay = (MOD & 2) != 0, kWide = sizeof(T) == 4;
    float unit, in, out, slope;
    __device__ __forceinline__ Score(float scale, float cap, float slope_) {
        unit = scale * kScoreUnit;
        in = kHasCap ? (kWide ? scale / cap : 2.f * kScoreUnit * scale / cap) : 0.f;
        out = cap * kScoreUnit;
        slope = slope_ * kScoreUnit;
    }
    __device__ __forceinline__ float r(float s) const { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * in)); }
    // x of an inner product s at distance `dist`; `grad` gets the derivative by scale * s, a quarter of it for 16-bit data.  It lies
    // in [0, 1], also where s is NaN: the masks of the backward pass come before it, and zero times NaN would undo them.  (That is
    // the clamp of the instruction which forms it and costs nothing; the masks behind it took 2 % of a step with capped scores.)
    __device__ __forceinline__ float operator()(float s, float dist, float &grad) const {
        float x;
        if constexpr (!kHasCap) x = s * unit;
        else if constexpr (!kWide) {
            const float a = r(s);
            x = __builtin_fmaf(a, -2.f * out, out);
            grad = __builtin_amdgcn_fmed3f(__builtin_fmaf(-a, a, a), 0.f, 1.f);
        } else {
            const float u = s * in, w = u * u;
            const float e = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.f * kScoreUnit * u));
            const float near = u * (1.f + w * (-1.f / 3 + w * (2.f / 15 + w * (-17.f / 315 + w * (62.f / 2835)))));
            const float t = __builtin_fabsf(u) < 0.25f ? near : 1.f - 2.f * e;
            x = t * out;
            grad = __builtin_amdgcn_fmed3f(__builtin_fmaf(-t, t, 1.f), 0.f, 1.f);
        }
        if constexpr (kHasDecay) x = __builtin_fmaf(-slope, __builtin_fabsf(dist), x);
        return x;
    }
    static constexpr float kGrad = kHasCap && !kWide ? 4.f : 1.f;   // what `grad` leaves to the end
};

// Nothing is moved across it: left to itself, the compiler reads every fragment right before its use and waits for it.
#define FLK_KEEP_ORDER() __builtin_amdgcn_sched_barrier(0)

// Which of a tile's 64 places this lane's row (or key) sees, one bit each.  Bit 8 g + 4 half + i of a block of 32 belongs to
// accumulator register 4 g + i, so the mask is shifted by 4 half once and every register asks for a fixed bit.
struct Seen {
    unsigned w[2];
    // all ones where register r of block kb is seen
    __device__ __forceinline__ int bits(int kb, int r) const { return (int)(w[kb] << (31 - (8 * (r >> 2) + (r & 3)))) >> 31; }
    __device__ __forceinline__ float or_inf(float x, int kb, int r) const {        // x, or -inf where it is hidden
        const int m = bits(kb, r);
        return __builtin_bit_cast(float, (__builtin_bit_cast(int, x) & m) | ((int)0xff800000 & ~m));
    }
    __device__ __forceinline__ float or_zero(float x, int kb, int r) const { return __builtin_bit_cast(float, __builtin_bit_cast(int, x) & bits(kb, r)); }
};
// a b, and zero where a is zero, also if b is an infinity or a NaN
__device__ __forceinline__ float times_or_zero(float a, float b) {
    float c;
    asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(c) : "v"(a), "v"(b));
    return c;
}
__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }
// The places whose id (place l's in lane l) is this lane's: one round for every different id among the lanes, which are few.
__device__ __forceinline__ uint64_t same_id(int place_id, int id) {
    uint64_t m = 0, todo = __ballot(id >= 0);
    while (todo != 0) {
        const int now = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        const uint64_t at = __ballot(place_id == now);
        const bool mine = id == now;
        m = mine ? at : m;
        todo &= ~__ballot(mine);
    }
    return m;
}
__device__ __forceinline__ Seen seen_from(uint64_t m) {
    m >>= 4 * (threadIdx.x >> 5 & 1);
    return {{(unsigned)m, (unsigned)(m >> 32)}};
}

// What the values that clean() took from a tile (its first `n` rows) do to the rows that see them: each, read again from memory, times
// `weight` is added to its column.  With 1 an infinity stays one, however small its weight (0 times it would be a NaN); with 0 it
// gives the NaN of weights that are zero whenever they are finite.  Rare, and not made to be fast; called with copies, so that the
// output stays in registers elsewhere.
template <typename T, int TK, int DB>
__device__ __noinline__ void spread_nonfinite(const T *rows, int64_t stride, int n, int d, Seen seen, float weight, fx16 *o) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const unsigned w[2] = {(unsigned)__shfl((int)seen.w[0], lane & 31, 64), (unsigned)__shfl((int)seen.w[1], lane & 31, 64)};  // not shifted
    for (int place = 0; place < min(n, TK); place++) {
        const T *row = rows + place * stride;
        bool bad = false;
        for (int c = lane; c < d; c += 64) bad |= !(__builtin_fabsf((float)row[c]) < kInf);
        if (!__any(bad)) continue;
        const bool mine = (place < 32 ? w[0] : w[1]) >> (place & 31) & 1;
        for (int db = 0; db < DB; db++)
            for (int r = 0; r < 16; r++) {
                const int c = 32 * db + 8 * (r >> 2) + 4 * half + (r & 3);
                const float v = c < d ? (float)row[c] : 0.f;
                if (mine && !(__builtin_fabsf(v) < kInf)) o[db][r] += v * weight;
            }
    }
}

// Columns of a gradient that are NaN because a value which is not finite stands in them, in a row of the other operand that this row
// sees: its weight is zero whenever it is finite itself.  A product with such values would reach the rows that hide them too, so it
// runs on zeros in their place (clean_block) and the columns are kept here, as bits in LDS: 32 rows of a wave, whose lanes of the first half
// write their own row's bits.
template <int DP> struct Spoilt {
    unsigned row[DP / 32];
    __device__ __forceinline__ void clear() {
        if ((threadIdx.x & 63) < 32) {
#pragma unroll
            for (int i = 0; i < DP / 32; i++) row[i] = 0;
        }
    }
    // the first `n` rows of a tile of the other operand, in memory
    template <typename T> __device__ __forceinline__ void note(const T *rows, int64_t stride, int n, int d, const Seen &seen) {
        const int lane = threadIdx.x & 63;
#pragma unroll 1
        for (int place = 0; place < n; place++) {
            const bool mine = lane < 32 && ((place < 32 ? seen.w[0] : seen.w[1]) >> (place & 31) & 1);   // (not shifted in this half)
#pragma unroll 1
            for (int c0 = 0; c0 < d; c0 += 64) {
                const int c = c0 + lane;
                const uint64_t bad = __ballot(c < d && !(__builtin_fabsf((float)rows[place * stride + min(c, d - 1)]) < kInf));
                if (bad == 0 || !mine) continue;
                row[c0 / 32] |= (unsigned)bad;
                if (c0 + 32 < DP) row[c0 / 32 + 1] |= (unsigned)(bad >> 32);
            }
        }
    }
    // `x`, the sums of this lane's row
    __device__ __forceinline__ void mark(fx16 *x) const {
        const int half = threadIdx.x >> 5 & 1;
#pragma unroll
        for (int db = 0; db < DP / 32; db++) {
            const unsigned w = row[db] >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; r++) x[db][r] = w >> (8 * (r >> 2) + (r & 3)) & 1 ? __builtin_nanf("") : x[db][r];
        }
    }
};

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

__device__ __forceinline__ float wave_maxf(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}

// smallest and largest document id of positions [lo, hi), a padding position counting as -1; (0, -1) if there is none
__device__ __forceinline__ int2 doc_span(const int2 *range, int lo, int hi) {
    int2 s = {0x7fffffff, -1};
    for (int b = lo / kDocBlock; b * kDocBlock < hi; b++) { s.x = min(s.x, range[b].x); s.y = max(s.y, range[b].y); }
    return s;
}
__device__ __forceinline__ bool docs_meet(int2 a, int2 b) { return a.y >= 0 && b.y >= 0 && a.x <= b.y && b.x <= a.y; }
__device__ __forceinline__ bool docs_same(int2 a, int2 b) { return a.x >= 0 && a.x == a.y && a.x == b.x && a.x == b.y; }

// The tiles a workgroup visits, in rising order, 64 at a time: lane t looks at tile base + t.  `whole`: no row of the
// workgroup needs a mask there; `full`, `skip`: this wave's rows need none, or see nothing.
struct TileWalk {
    int base, end;
    uint64_t todo, whole, full, skip;
    bool is_whole, is_full, is_skip;
    __device__ __forceinline__ void start(int lo, int hi) { base = lo - 64; end = hi; todo = 0; }
    template <typename Look> __device__ __forceinline__ int next(Look look) {
        while (todo == 0) {
            base += 64;
            if (base >= end) return -1;
            const int t = base + (int)(threadIdx.x & 63);
            bool want = t < end, w = false, f = false, s = false;
            if (want) look(t, want, w, f, s);
            todo = __ballot(want);
            whole = __ballot(w);
            full = __ballot(f);
            skip = __ballot(s);
        }
        const int i = __builtin_ctzll(todo);
        todo &= todo - 1;
        is_whole = whole >> i & 1;
        is_full = full >> i & 1;
        is_skip = skip >> i & 1;
        return base + i;
    }
};

constexpr int kCachedKeys = 32;            // keys of a wave's tile

struct CachedArgs {
    const void *q, *k, *v;
    void *out;
    AttnStride qs, ks, vs;                 // q: [b][t][hq][d]
    const int *lengths;
    const float *slopes;
    float *part_o, *part_ml;               // parts of several workgroups: [row][split][dv] and [row][split][2]
    int b, t, capacity, hq, hk, group, d, dv_d, splits, blocks_r;
    int waves;                             // of a workgroup: 4, or 8 where their tiles fit into LDS
    float scale, cap;
    int vec;
};

// What the kernels look like from a launcher (attention.hip); one source per element type instantiates them.
template <typename T> int launch_attention_fwd(const AttnArgs &a, int dp, hipStream_t st);
template <typename T> int launch_attention_dq(const AttnArgs &a, int dp, hipStream_t st);
template <typename T> int launch_attention_dkv(const AttnArgs &a, int dp, hipStream_t st);
template <typename T> int launch_attention_cached(const CachedArgs &a, int dp, hipStream_t st);

inline int score_kind(float scale, float cap, const float *slopes) {
    return (cap > 0.f ? kCap : kPlain) | (slopes != nullptr || !(scale > 0.f) ? kDecay : 0);
}
#define FLK_ATTN_KIND(KERNEL, DP, GRID)                                                                            \
    {                                                                                                              \
        if (kind == kPlain) hipLaunchKernelGGL((KERNEL<T, DP, kPlain>), GRID, dim3(kAttnThreads), 0, st, a);       \
        else if (kind == kCap) hipLaunchKernelGGL((KERNEL<T, DP, kCap>), GRID, dim3(kAttnThreads), 0, st, a);      \
        else if (kind == kDecay) hipLaunchKernelGGL((KERNEL<T, DP, kDecay>), GRID, dim3(kAttnThreads), 0, st, a);  \
        else hipLaunchKernelGGL((KERNEL<T, DP, kCapDecay>), GRID, dim3(kAttnThreads), 0, st, a);                   \
    }
#define FLK_ATTN_LAUNCH_KIND(KERNEL, GRID)                         \
    {                                                              \
        if (dp == 32) FLK_ATTN_KIND(KERNEL, 32, GRID)              \
        else if (dp == 64) FLK_ATTN_KIND(KERNEL, 64, GRID)         \
        else if (dp == 96) FLK_ATTN_KIND(KERNEL, 96, GRID)         \
        else FLK_ATTN_KIND(KERNEL, 128, GRID)                      \
        FLK_LAUNCH_CHECK(#KERNEL);                                 \
    }
#define FLK_ATTN_LAUNCH(KERNEL, GRID)                              \
    const int kind = score_kind(a.scale, a.cap, a.slopes);         \
    FLK_ATTN_LAUNCH_KIND(KERNEL, GRID)

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
