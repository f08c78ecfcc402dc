// extern "C" entry points of the attention operators: argument checks, workspaces, launch plans, and the small kernels beside
// them (document spans, sums of parts).
#include "attention_common.h"

namespace flk {

// Smallest and largest document id of every kDocBlock positions, a padding position (a negative id) counting as -1; and the ids
// themselves, row after row from a multiple of 16 bytes on, -1 for padding and past the end.
__global__ void __launch_bounds__(kAttnThreads) attention_doc_kernel(const int *docs, int64_t docs_b, int n, int blocks, int64_t total, int2 *out,
                                                                     int *ids) {
    const int64_t i = (int64_t)blockIdx.x * (kAttnThreads / kDocBlock) + threadIdx.x / kDocBlock;
    const int64_t b = (i < total ? i : 0) / blocks;
    const int pos = (int)((i < total ? i : 0) % blocks) * kDocBlock + threadIdx.x % kDocBlock;
    const int id = pos < n ? max(docs[b * docs_b + pos], -1) : -1;
    int lo = pos < n ? id : 0x7fffffff, hi = id;
#pragma unroll
    for (int o = kDocBlock / 2; o > 0; o >>= 1) { lo = min(lo, __shfl_xor(lo, o, 64)); hi = max(hi, __shfl_xor(hi, o, 64)); }
    if (i >= total) return;
    ids[i * kDocBlock + threadIdx.x % kDocBlock] = id;
    if (threadIdx.x % kDocBlock == 0) out[i] = {lo, hi};
}

// dslopes[h]: the workgroups' sums, in double and in a fixed order (their terms cancel)
__global__ void __launch_bounds__(kAttnThreads) attention_dslopes_kernel(const float *part, int64_t n, float *out) {
    __shared__ double lds[kAttnThreads];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kAttnThreads) s += (double)part[blockIdx.x * n + i];
    lds[threadIdx.x] = s;
    __syncthreads();
    for (int o = kAttnThreads / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) lds[threadIdx.x] += lds[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[blockIdx.x] = (float)lds[0];
}

// out, rest and lse from the parts of the forward kernel, one thread a value
template <typename T> __global__ void __launch_bounds__(kAttnThreads) attention_parts_kernel(AttnArgs p) {
    const int64_t rows = (int64_t)p.b * p.sq * p.hq, i = (int64_t)blockIdx.x * kAttnThreads + threadIdx.x;
    if (i >= rows * p.dv_d) return;
    const int64_t row = i / p.dv_d, c = i % p.dv_d;
    float top = -kInf;
    for (int k = 0; k < p.parts; k++) top = fmaxf(top, p.part_ml[(k * rows + row) * 2]);
    float x = 0.f, l = 0.f;
    for (int k = 0; k < p.parts; k++) {
        const float m = p.part_ml[(k * rows + row) * 2], lk = p.part_ml[(k * rows + row) * 2 + 1];
        if (m == -kInf && lk == 0.f) continue;                     // saw nothing
        const float a = m == -kInf ? 1.f : __builtin_amdgcn_exp2f(m - top);
        x += a * p.part_o[(k * rows + row) * p.dv_d + c];
        l += a * lk;
    }
    const float y = l == 0.f ? 0.f : x / l;
    const T z = (T)y;
    ((T *)p.o)[i] = z;
    if (p.rest != nullptr) ((T *)p.rest)[i] = (T)(y - (float)z);
    if (c == 0 && p.lse != nullptr) {
        const int64_t h = row % p.hq, s = row / p.hq % p.sq, b = row / p.hq / p.sq;
        p.lse[(b * p.hq + h) * p.sq + s] = l == 0.f ? -kInf : top * kLn2 + __logf(l);
    }
}

// dq, dk and dv from their parts
struct JoinArgs { const float *part[3]; void *to[3]; int64_t n[3]; int parts[3]; };
template <typename T> __global__ void __launch_bounds__(kAttnThreads) attention_join_kernel(JoinArgs p) {
    int64_t i = (int64_t)blockIdx.x * kAttnThreads + threadIdx.x;
#pragma unroll
    for (int k = 0; k < 3; k++) {
        if (i >= 0 && i < p.n[k]) {
            float s = 0.f;
            for (int j = 0; j < p.parts[k]; j++) s += p.part[k][j * p.n[k] + i];
            ((T *)p.to[k])[i] = (T)s;
        }
        i -= p.n[k];
    }
}

constexpr int64_t kMaxPositions = (int64_t)1 << 28;
constexpr int64_t kMaxGrid = 0x7fffffff;
static int elem_size(int dtype) { return dtype == FLK_F32 ? 4 : 2; }
static bool attn_dtype(int dtype) { return dtype == FLK_F32 || dtype == FLK_F16 || dtype == FLK_BF16; }
static int padded_d(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128; }
static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
static bool rows_aligned(const void *p, const AttnStride &s, int64_t d, int es) {
    const int64_t e = 16 / es;
    if (s.s > ((int64_t)1 << 23) || s.s < 0) return false;        // a tile's offsets are 32 bits wide
    return aligned16(p) && s.b % e == 0 && s.s % e == 0 && s.h % e == 0 && d % e == 0;
}

// document spans, then ids
static int64_t doc_bytes(int64_t b, int64_t sk) {
    const int64_t n = b * cdiv(sk, kDocBlock);
    return align256((size_t)n * sizeof(int2)) + align256((size_t)n * kDocBlock * 4);
}
static void place_docs(AttnArgs &a, void *ws) {
    a.doc_range = (int2 *)ws;
    a.doc_ids = (int *)((char *)ws + align256((size_t)a.b * a.doc_blocks * sizeof(int2)));
}

// Workgroups among which a tile of 128 rows divides its tiles of keys (or queries).  One wave's way through them all takes its
// time however few workgroups there are, so where they do not fill the chip they are made shorter: up to 512 in all, none
// with less than eight tiles (four of float, which take four times as long).  The parts are written in float and read again,
// so there are no more than eight.
// (Float, 2 x 8 heads of 80, 1000 positions: forward 116 -> 78 us, backward 379 -> 222; bf16, 8 heads of 128, 2048 positions:
// forward 53 -> 50, backward 161 -> 129.)
static int parts_for(int64_t groups, int64_t keys, int dtype) {
    const int64_t most = elem_size(dtype) == 4 ? cdiv(keys, 32) / 4 : cdiv(keys, 64) / 8;
    int64_t n = groups > 0 ? 512 / groups : 1;
    if (n > most) n = most;
    return (int)(n < 1 ? 1 : n > 8 ? 8 : n);
}

struct AttnSizes { int64_t doc_blocks, docs, sq_pad, stats, sizes, bad, slopes, dq, dkv; int parts, head_parts, row_parts; };
static AttnSizes attn_sizes(int64_t b, int64_t sq, int64_t sk, int64_t hq, int64_t hk, int64_t d, int64_t dv, bool docs, bool slopes, int dtype) {
    AttnSizes z = {};
    z.doc_blocks = cdiv(sk, kDocBlock);
    z.docs = docs ? doc_bytes(b, sk) : 0;
    z.sq_pad = cdiv(sq, kAttnRows) * kAttnRows;
    z.stats = align256((size_t)(b * hq * z.sq_pad) * 12);
    z.sizes = dtype == FLK_F16 ? align256((size_t)(b * hq * z.sq_pad / 32) * 8) : 0;
    z.bad = align256((size_t)(b * hq * z.sq_pad / 32));
    z.slopes = slopes ? align256((size_t)(b * hq * cdiv(sq, kAttnRows)) * 4) : 0;
    // (the slopes' gradient is a product of two of a row's sums, so their rows are not divided)
    z.parts = slopes ? 1 : parts_for(b * hq * cdiv(sq, kAttnRows), sk, dtype);
    z.dq = z.parts > 1 ? align256((size_t)z.parts * b * sq * hq * d * 4) : 0;
    // dk / dv: the query heads that share the key head are divided first, then the tiles of queries
    const int64_t groups = b * hk * cdiv(sk, kAttnRows), group = hk > 0 ? hq / hk : 1;
    z.head_parts = 1;
    if (groups > 0 && groups < 512) z.head_parts = (int)(cdiv(512, groups) < group ? cdiv(512, groups) : group);
    if (z.head_parts < 1) z.head_parts = 1;
    if (z.head_parts > 8) z.head_parts = 8;
    z.row_parts = parts_for(groups * z.head_parts, sq, dtype);
    if (z.row_parts * z.head_parts > 8) z.row_parts = 8 / z.head_parts;
    z.dkv = z.head_parts * z.row_parts > 1 ? align256((size_t)z.head_parts * z.row_parts * b * sk * hk * (d + dv) * 4) : 0;
    return z;
}

static int attn_check(const char *what, int64_t b, int64_t sq, int64_t sk, int64_t hq, int64_t hk, int64_t d, int64_t dv, double scale, double softcap,
                      int causal, const int *prefix, const int *docs, int dtype) {
    if (b < 0 || sq < 0 || sk < 0 || hq < 1 || hk < 1 || d < 1 || dv < 1) return fail(FLK_EINVAL, "%s: bad shape", what);
    if (hq % hk != 0) return fail(FLK_EINVAL, "%s: %lld query heads cannot share %lld key heads evenly", what, (long long)hq, (long long)hk);
    if (!attn_dtype(dtype)) return fail(FLK_EINVAL, "%s: unknown dtype %d", what, dtype);
    if (d > kAttnMaxD || dv > kAttnMaxD) return fail(FLK_EUNSUPPORTED, "%s: heads of more than %d values", what, kAttnMaxD);
    if (sq > kMaxPositions || sk > kMaxPositions) return fail(FLK_EUNSUPPORTED, "%s: more than %lld positions", what, (long long)kMaxPositions);
    if (!(softcap >= 0.0)) return fail(FLK_EINVAL, "%s: softcap must not be negative", what);
    const double max_cap = dtype == FLK_F32 ? kMaxCap : kMaxCap16;
    if (softcap > 0.0 && (softcap < kMinCap || softcap > max_cap))
        return fail(FLK_EUNSUPPORTED, "%s: softcap of %g (%g to %g)", what, softcap, kMinCap, max_cap);
    if (!(scale >= -kMaxScale && scale <= kMaxScale)) return fail(FLK_EUNSUPPORTED, "%s: scale of %g (at most %g)", what, scale, kMaxScale);
    if (prefix != nullptr && !causal) return fail(FLK_EINVAL, "%s: a prefix belongs to a causal mask", what);
    if (docs != nullptr && sq > sk) return fail(FLK_EINVAL, "%s: documents need every query to stand at a key's position", what);
    if (b > 0 && (hq > kMaxGrid / b || b * hq * cdiv(sq > sk ? sq : sk, kAttnRows) > kMaxGrid))
        return fail(FLK_EUNSUPPORTED, "%s: too many rows for one launch", what);
    return FLK_OK;
}

static int launch_docs(const AttnArgs &a, hipStream_t st) {
    const int64_t total = (int64_t)a.b * a.doc_blocks;
    if (a.docs == nullptr || total == 0) return FLK_OK;
    hipLaunchKernelGGL(attention_doc_kernel, dim3((unsigned)cdiv(total, kAttnThreads / kDocBlock)), dim3(kAttnThreads), 0, st, a.docs,
                       a.docs_b, a.sk, a.doc_blocks, total, a.doc_range, a.doc_ids);
    FLK_LAUNCH_CHECK("attention_doc_kernel");
    return FLK_OK;
}

template <typename T> static int attention_backward_impl(AttnArgs &a, int dp, float *dslopes, hipStream_t st) {
    int rc = FLK_OK;
    if ((int64_t)a.b * a.sq > 0 && (rc = launch_attention_dq<T>(a, dp, st)) != FLK_OK) return rc;
    if (dslopes != nullptr) {
        hipLaunchKernelGGL(attention_dslopes_kernel, dim3((unsigned)a.hq), dim3(kAttnThreads), 0, st, a.dslopes_part,
                           (int64_t)a.b * cdiv(a.sq, kAttnRows), dslopes);
        FLK_LAUNCH_CHECK("attention_dslopes_kernel");
    }
    JoinArgs join = {};
    if (a.dq != nullptr && a.parts > 1) {
        join.part[0] = a.dq_part; join.to[0] = a.dq; join.n[0] = (int64_t)a.b * a.sq * a.hq * a.d; join.parts[0] = a.parts;
    }
    if (a.dk != nullptr && (int64_t)a.b * a.sk > 0) {
        if ((rc = launch_attention_dkv<T>(a, dp, st)) != FLK_OK) return rc;
        const int splits = a.head_parts * a.row_parts;
        if (splits > 1) {
            const int64_t keys = (int64_t)a.b * a.sk * a.hk, nk = keys * a.d;
            join.part[1] = a.dkv_part; join.to[1] = a.dk; join.n[1] = nk; join.parts[1] = splits;
            join.part[2] = a.dkv_part + splits * nk; join.to[2] = a.dv; join.n[2] = keys * a.dv_d; join.parts[2] = splits;
        }
    }
    const int64_t n = join.n[0] + join.n[1] + join.n[2];
    if (n == 0) return FLK_OK;
    hipLaunchKernelGGL((attention_join_kernel<T>), dim3((unsigned)cdiv(n, kAttnThreads)), dim3(kAttnThreads), 0, st, join);
    FLK_LAUNCH_CHECK("attention_join_kernel");
    return FLK_OK;
}

template <typename T> static int attention_forward_impl(AttnArgs &a, int dp, hipStream_t st) {
    const int rc = launch_attention_fwd<T>(a, dp, st);
    if (rc != FLK_OK || a.parts == 1) return rc;
    const int64_t n = (int64_t)a.b * a.sq * a.hq * a.dv_d;
    hipLaunchKernelGGL((attention_parts_kernel<T>), dim3((unsigned)cdiv(n, kAttnThreads)), dim3(kAttnThreads), 0, st, a);
    FLK_LAUNCH_CHECK("attention_parts_kernel");
    return FLK_OK;
}

// forward: the documents' spans and ids, then the parts of out and of the rows' maxima and sums
struct FwdSizes { int64_t docs, o, ml; int parts; };
static FwdSizes fwd_sizes(int64_t b, int64_t sq, int64_t sk, int64_t hq, int64_t dv, bool docs, int dtype) {
    FwdSizes z = {};
    z.docs = docs ? doc_bytes(b, sk) : 0;
    z.parts = parts_for(b * hq * cdiv(sq, kAttnRows), sk, dtype);
    if (z.parts > 1) {
        z.o = align256((size_t)z.parts * b * sq * hq * dv * 4);
        z.ml = align256((size_t)z.parts * b * sq * hq * 8);
    }
    return z;
}

// Workgroups the keys of a sequence are divided over: as many as run at once, since every part more is written and added again and
// a few workgroups more would be a second round (11 sequences of 8000 keys, 8 key heads of 128: 77 us with 440, 92 with 528; 7 of 16 000 floats,
// 12 heads of 64: 149 with 504, 198 with 588; but 40 of 4000, 8 heads of 128: 145 with 320, 140 with 640), and none with less than four
// tiles for each of four waves at the cache's capacity.  At once run two workgroups of four waves on a compute
// unit; heads above 64 values do better with one of eight (cached_waves), where that leaves few units idle (bf16, heads of 128: 4 key
// heads and 121 900 keys 52.8 us so, 58.5 with two of four; 8 sequences of 8000 keys, 8 key heads, 47.6 and 49.3.  Heads of 64: 2
// sequences of 32 000 keys, 8 key heads, 30.6 and 28.9).
// Less than four parts do not make up for the second kernel.  Where the sequences alone fill the chip,
// parts of at most 4096 keys (four at most) even out their lengths (64 of up to 16384 keys: 426 us with 4 parts, 474 undivided;
// of up to 1024: 39 us with 2, 33 undivided).
static int cached_splits(int64_t b, int64_t t, int64_t capacity, int64_t hq, int64_t hk, int64_t dv) {
    const int64_t groups = b * hk * cdiv(t * (hq / hk), 32);
    int64_t most = cdiv(capacity, 4 * 4 * kCachedKeys);
    if (most < 4) most = 1;
    int64_t n = groups > 0 ? 512 / groups : 1;
    if (dv > 64 && groups > 0 && 256 / groups * groups >= 240) n = 256 / groups;
    const int64_t even = capacity / 4096 < 4 ? capacity / 4096 : 4;
    if (b > 1 && n < even) n = even;
    if (n > most) n = most;
    return (int)(n < 1 ? 1 : n > 256 ? 256 : n);
}

// Waves of a workgroup.  A wave's way through its tiles is what a call takes as long as there is a compute unit for every workgroup, so
// eight halve it (bf16, 8 key heads of 128, 1000 keys: one sequence 24.5 us with four waves, 16.7 with eight; 32 sequences 26.9 and
// 25.5); with more workgroups four leave room for two of them on a unit (64 sequences: 45.0 us, and 47.9 with eight).  Up to four
// tiles give the others nothing to do (100 keys: 5.5 us, and 5.8 with eight).
static int cached_waves(int64_t workgroups, int64_t capacity) { return workgroups <= 256 && capacity > 4 * kCachedKeys ? 8 : 4; }

}  // namespace flk

using namespace flk;

#define FLK_BY_TYPE(dtype, CALL)                       \
    (dtype == FLK_F32 ? CALL(float) : dtype == FLK_F16 ? CALL(f16_t) : CALL(bf16_t))

extern "C" {

int64_t flk_attention_max_d(int dtype) { return attn_dtype(dtype) ? kAttnMaxD : 0; }

size_t flk_attention_workspace_bytes(int64_t b, int64_t sq, int64_t sk, int64_t hq, int64_t dv, int with_documents, int dtype) {
    if (b < 0 || sq < 0 || sk < 0 || sq > kMaxPositions || sk > kMaxPositions || hq < 1 || dv < 1 || !attn_dtype(dtype)) return 0;
    const FwdSizes z = fwd_sizes(b, sq, sk, hq, dv, with_documents != 0, dtype);
    return (size_t)(z.docs + z.o + z.ml);
}

int flk_attention(const void *q, int64_t q_b, int64_t q_s, int64_t q_h, const void *k, int64_t k_b, int64_t k_s, int64_t k_h,
                  const void *v, int64_t v_b, int64_t v_s, int64_t v_h, int64_t b, int64_t sq, int64_t sk, int64_t hq, int64_t hk,
                  int64_t d, int64_t dv, double scale, double softcap, const float *slopes, int causal, const int *prefix,
                  const int *documents, int64_t documents_b, void *out, void *rest, float *lse, int dtype, void *workspace,
                  size_t workspace_bytes, void *stream) {
    fail(FLK_OK, "%s", "");
    int rc = attn_check("flk_attention", b, sq, sk, hq, hk, d, dv, scale, softcap, causal, prefix, documents, dtype);
    if (rc != FLK_OK || b * sq == 0) return rc;
    if (q == nullptr || out == nullptr || (sk > 0 && (k == nullptr || v == nullptr))) return fail(FLK_EINVAL, "flk_attention: null pointer");
    const FwdSizes z = fwd_sizes(b, sq, sk, hq, dv, documents != nullptr, dtype);
    const size_t need = (size_t)(z.docs + z.o + z.ml);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(FLK_ENOMEM, "workspace of %zu bytes given, %zu needed", workspace_bytes, need);
    AttnArgs a = {};
    a.q = q; a.k = k; a.v = v; a.o = out; a.rest = dtype == FLK_F32 ? nullptr : rest; a.lse = lse;
    a.qs = {q_b, q_s, q_h}; a.ks = {k_b, k_s, k_h}; a.vs = {v_b, v_s, v_h};
    a.b = (int)b; a.sq = (int)sq; a.sk = (int)sk; a.hq = (int)hq; a.hk = (int)hk; a.group = (int)(hq / hk); a.d = (int)d; a.dv_d = (int)dv;
    a.scale = (float)scale; a.cap = (float)softcap; a.slopes = slopes; a.causal = causal != 0; a.prefix = prefix;
    a.docs = documents; a.docs_b = documents_b; a.doc_blocks = (int)cdiv(sk, kDocBlock);
    a.parts = z.parts;
    char *ws = (char *)workspace;
    place_docs(a, ws); ws += z.docs;
    a.part_o = (float *)ws; ws += z.o;
    a.part_ml = (float *)ws;
    const int es = elem_size(dtype);
    a.vec = rows_aligned(q, a.qs, d, es) && rows_aligned(k, a.ks, d, es);
    a.vec_v = rows_aligned(v, a.vs, dv, es) && aligned16(out) && aligned16(a.rest);
    hipStream_t st = (hipStream_t)stream;
    if ((rc = launch_docs(a, st)) != FLK_OK) return rc;
    const int dp = padded_d(d > dv ? d : dv);
#define FLK_CALL(T) attention_forward_impl<T>(a, dp, st)
    return FLK_BY_TYPE(dtype, FLK_CALL);
#undef FLK_CALL
}

size_t flk_attention_backward_workspace_bytes(int64_t b, int64_t sq, int64_t sk, int64_t hq, int64_t hk, int64_t d, int64_t dv,
                                              int with_slopes, int with_documents, int dtype) {
    if (b < 0 || sq < 0 || sk < 0 || hq < 1 || hk < 1 || d < 1 || dv < 1 || hq % hk != 0 || sq > kMaxPositions || sk > kMaxPositions || !attn_dtype(dtype))
        return 0;
    const AttnSizes z = attn_sizes(b, sq, sk, hq, hk, d, dv, with_documents != 0, with_slopes != 0, dtype);
    return (size_t)(z.docs + z.stats + z.sizes + z.bad + z.slopes + z.dq + z.dkv);
}

int flk_attention_backward(const void *q, int64_t q_b, int64_t q_s, int64_t q_h, const void *k, int64_t k_b, int64_t k_s, int64_t k_h,
                           const void *v, int64_t v_b, int64_t v_s, int64_t v_h, const void *out, const void *rest, const float *lse, const void *dout,
                           int64_t do_b, int64_t do_s, int64_t do_h, int64_t b, int64_t sq, int64_t sk, int64_t hq, int64_t hk, int64_t d,
                           int64_t dv, double scale, double softcap, const float *slopes, int causal, const int *prefix,
                           const int *documents, int64_t documents_b, void *dq, void *dk, void *dv_out, float *dslopes, int dtype,
                           void *workspace, size_t workspace_bytes, void *stream) {
    fail(FLK_OK, "%s", "");
    int rc = attn_check("flk_attention_backward", b, sq, sk, hq, hk, d, dv, scale, softcap, causal, prefix, documents, dtype);
    if (rc != FLK_OK) return rc;
    if ((dk == nullptr) != (dv_out == nullptr)) return fail(FLK_EINVAL, "flk_attention_backward: dk and dv come together");
    if (dslopes != nullptr && slopes == nullptr) return fail(FLK_EINVAL, "flk_attention_backward: no slopes to differentiate");
    if ((b * sq > 0 && (q == nullptr || out == nullptr || lse == nullptr || dout == nullptr)) || (b * sk > 0 && (k == nullptr || v == nullptr)))
        return fail(FLK_EINVAL, "flk_attention_backward: null pointer");
    const AttnSizes z = attn_sizes(b, sq, sk, hq, hk, d, dv, documents != nullptr, dslopes != nullptr, dtype);
    const size_t need = (size_t)(z.docs + z.stats + z.sizes + z.bad + z.slopes + z.dq + z.dkv);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(FLK_ENOMEM, "workspace of %zu bytes given, %zu needed", workspace_bytes, need);
    AttnArgs a = {};
    a.q = q; a.k = k; a.v = v; a.out = out; a.rest = dtype == FLK_F32 ? nullptr : (void *)rest; a.dout = dout; a.lse = (float *)lse; a.dq = dq; a.dk = dk; a.dv = dv_out;
    a.qs = {q_b, q_s, q_h}; a.ks = {k_b, k_s, k_h}; a.vs = {v_b, v_s, v_h};
    a.dos = {do_b, do_s, do_h}; a.sq_pad = z.sq_pad;
    a.b = (int)b; a.sq = (int)sq; a.sk = (int)sk; a.hq = (int)hq; a.hk = (int)hk; a.group = (int)(hq / hk); a.d = (int)d; a.dv_d = (int)dv;
    a.scale = (float)scale; a.cap = (float)softcap; a.slopes = slopes; a.causal = causal != 0; a.prefix = prefix;
    a.docs = documents; a.docs_b = documents_b; a.doc_blocks = (int)z.doc_blocks;
    a.parts = z.parts; a.head_parts = z.head_parts; a.row_parts = z.row_parts;
    char *ws = (char *)workspace;
    place_docs(a, ws); ws += z.docs;
    a.stats = (float *)ws; ws += z.stats;
    a.sizes = (float2 *)ws; ws += z.sizes;
    a.bad_rows = (unsigned char *)ws; ws += z.bad;
    a.dslopes_part = dslopes != nullptr ? (float *)ws : nullptr; ws += z.slopes;
    a.dq_part = (float *)ws; ws += z.dq;
    a.dkv_part = (float *)ws;
    const int es = elem_size(dtype);
    a.vec = rows_aligned(q, a.qs, d, es) && rows_aligned(k, a.ks, d, es) && aligned16(dq) && aligned16(dk);
    a.vec_v = rows_aligned(v, a.vs, dv, es) && rows_aligned(dout, a.dos, dv, es) && aligned16(out) && aligned16(a.rest) && aligned16(dv_out);
    hipStream_t st = (hipStream_t)stream;
    if ((rc = launch_docs(a, st)) != FLK_OK) return rc;
    const int dp = padded_d(d > dv ? d : dv);
#define FLK_CALL(T) attention_backward_impl<T>(a, dp, dslopes, st)
    return FLK_BY_TYPE(dtype, FLK_CALL);
#undef FLK_CALL
}

size_t flk_attention_cached_workspace_bytes(int64_t b, int64_t t, int64_t capacity, int64_t hq, int64_t hk, int64_t dv) {
    if (b < 0 || t < 0 || capacity < 0 || hq < 1 || hk < 1 || dv < 1 || hq % hk != 0) return 0;
    const int64_t n = cached_splits(b, t, capacity, hq, hk, dv);
    return n > 1 ? align256((size_t)(b * t * hq * n * dv) * 4) + align256((size_t)(b * t * hq * n * 2) * 4) : 0;
}

int flk_attention_cached(const void *q, int64_t q_b, int64_t q_s, int64_t q_h, const void *k, int64_t k_b, int64_t k_s, int64_t k_h,
                         const void *v, int64_t v_b, int64_t v_s, int64_t v_h, const int *lengths, int64_t b, int64_t t,
                         int64_t capacity, int64_t hq, int64_t hk, int64_t d, int64_t dv, double scale, double softcap,
                         const float *slopes, void *out, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    fail(FLK_OK, "%s", "");
    int rc = attn_check("flk_attention_cached", b, t, capacity, hq, hk, d, dv, scale, softcap, 1, nullptr, nullptr, dtype);
    if (rc != FLK_OK || b * t == 0) return rc;
    if (q == nullptr || out == nullptr || lengths == nullptr || (capacity > 0 && (k == nullptr || v == nullptr)))
        return fail(FLK_EINVAL, "flk_attention_cached: null pointer");
    const int64_t n = cached_splits(b, t, capacity, hq, hk, dv);
    const size_t need = flk_attention_cached_workspace_bytes(b, t, capacity, hq, hk, dv);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(FLK_ENOMEM, "workspace of %zu bytes given, %zu needed", workspace_bytes, need);
    CachedArgs a = {};
    a.q = q; a.k = k; a.v = v; a.out = out;
    a.qs = {q_b, q_s, q_h}; a.ks = {k_b, k_s, k_h}; a.vs = {v_b, v_s, v_h};
    a.lengths = lengths; a.slopes = slopes;
    a.part_o = (float *)workspace;
    a.part_ml = (float *)((char *)workspace + (n > 1 ? align256((size_t)(b * t * hq * n * dv) * 4) : 0));
    a.b = (int)b; a.t = (int)t; a.capacity = (int)capacity; a.hq = (int)hq; a.hk = (int)hk; a.group = (int)(hq / hk); a.d = (int)d;
    a.dv_d = (int)dv; a.splits = (int)n; a.blocks_r = (int)cdiv(t * (hq / hk), 32); a.scale = (float)scale; a.cap = (float)softcap;
    const int64_t grid = b * hk * a.blocks_r * n;
    a.waves = cached_waves(grid, capacity);
    if (grid > kMaxGrid || b * t * hq > kMaxGrid) return fail(FLK_EUNSUPPORTED, "flk_attention_cached: too many rows for one launch");
    const int es = elem_size(dtype);
    a.vec = rows_aligned(q, a.qs, d, es) && rows_aligned(k, a.ks, d, es) && rows_aligned(v, a.vs, dv, es);
    hipStream_t st = (hipStream_t)stream;
    const int dp = padded_d(d > dv ? d : dv);
#define FLK_CALL(T) launch_attention_cached<T>(a, dp, st)
    return FLK_BY_TYPE(dtype, FLK_CALL);
#undef FLK_CALL
}

}  // extern "C"
