// Attention, forward: one pass over the keys with a running maximum and sum (gfx950).  Compiled once per element type.
//
// A workgroup owns 128 queries of one head, a wave 32 of them, with its queries and its 32 x d output in registers; tiles of
// keys and values go through LDS, the next one on its way while the present one is used.  The output is rescaled only when
// some row of the wave found a maximum well above the one in use.  Scores and probabilities never leave the registers.
#include "attention_common.h"

namespace flk {

// A maximum is taken over only when a row exceeds the present one by this much (in units of log 2): weights then lie below
// 2^kSlack, which every type holds, and most tiles after the first need no rescaling.
constexpr float kSlack = 6.f;
// ... and float16's lie between 2^14 for the largest and 2^-14, the last normal number, for one of 2^-22 of the maximum
template <typename T> constexpr float kLift = kNarrow<T> ? 8.f : 0.f;

template <typename T, int DP, int MOD>
__global__ void __launch_bounds__(kAttnThreads, (sizeof(T) == 2 && DP <= 64 ? 3 : 2)) attention_fwd_kernel(AttnArgs p) {
    typedef AttnType<T> AT;
    typedef typename AT::frag frag;
    typedef Tile<T, DP> TL;
    constexpr int TK = AT::kTile, KB = TK / 32, C = DP / AT::KS, DB = DP / 32, ST = 32 / AT::KS;
    typedef Feed<T, DP, TK> FD;
    constexpr int kTileBytes = TK * TL::RB;
    __shared__ __align__(16) char lds[4 * kTileBytes];
    __shared__ int lds_doc[8];
    __shared__ int lds_bad;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    // consecutive workgroups go to different XCDs: heads that share keys stay on one of them, the longest rows go first
    const int heads = p.b * p.hq, pairs = p.b * p.hk;
    const int hb = blockIdx.x % heads, tiles_q = (p.sq + kAttnRows - 1) / kAttnRows;
    const int tile_q = tiles_q - 1 - blockIdx.x / heads % tiles_q, part = blockIdx.x / heads / tiles_q;
    const int b = hb % pairs / p.hk, hk = hb % p.hk, h = hk * p.group + hb / pairs;
    const int off = p.sk - p.sq;
    const int i0 = tile_q * kAttnRows, row = i0 + wave * 32 + (lane & 31);
    const bool live = row < p.sq;
    const int pos = row + off, pos_lo = i0 + wave * 32 + off;
    const int pos_end = min(i0 + kAttnRows, p.sq) + off;           // behind the last position of the workgroup
    const Score<T, MOD> score(p.scale, p.cap, (MOD & kDecay) && p.slopes != nullptr ? p.slopes[h] : 0.f);
    constexpr bool kLate = MOD == kPlain || (MOD == kCap && sizeof(T) == 2);   // rising in s: the maximum is looked for before
    const int prefix = p.prefix != nullptr ? max(min(p.prefix[b], p.sk), 0) : 0;
    const int last = p.causal ? min(max(pos, prefix - 1), p.sk - 1) : p.sk - 1;   // last key this row sees

    const T *qrow = (const T *)p.q + b * p.qs.b + h * p.qs.h + (int64_t)row * p.qs.s;
    typename TL::Lane at_lane;
    at_lane.init();
    FD feed_k, feed_v;
    feed_k.init((const T *)p.k + b * p.ks.b + hk * p.ks.h, p.ks.s, p.d, p.vec);
    feed_v.init((const T *)p.v + b * p.vs.b + hk * p.vs.h, p.vs.s, p.dv_d, p.vec_v);
    frag qf[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        union { ux4 u; frag f; } x;
        x.u = load_chunk<T>(qrow, 2 * c + half, p.d, live, p.vec);
        qf[c] = x.f;
    }

    // documents: this row's id (negative: sees nothing) and the span of the wave's and of the workgroup's rows
    int id = 0;
    int2 span = {0, 0}, wg_span = {0, 0};
    const int2 *ranges = p.doc_range + (int64_t)b * p.doc_blocks;
    const int *ids = p.doc_ids + (int64_t)b * p.doc_blocks * kDocBlock;
    if (threadIdx.x == 0) lds_bad = -1;
    if (p.docs != nullptr) {
        const int raw = live ? ids[pos] : -1;
        span = {wave_min(raw), wave_max(raw)};
        if (lane == 0) { lds_doc[wave] = span.x; lds_doc[4 + wave] = span.y; }
        id = raw;
        __syncthreads();
        wg_span.x = min(min(lds_doc[0], lds_doc[1]), min(lds_doc[2], lds_doc[3]));
        wg_span.y = max(max(lds_doc[4], lds_doc[5]), max(lds_doc[6], lds_doc[7]));
    }
    const int key_end = p.causal ? max(min(pos_end, p.sk), prefix) : p.sk;
    TileWalk walk;
    const int64_t tiles_k = key_end > 0 ? (key_end + TK - 1) / TK : 0;
    walk.start((int)(tiles_k * part / p.parts), (int)(tiles_k * (part + 1) / p.parts));
    const auto look = [&](int t, bool &want, bool &whole, bool &full, bool &skip) {
        const int k0 = t * TK, k1 = k0 + TK;
        const bool inside = k1 <= p.sk, in_prefix = !p.causal || k1 <= prefix;
        whole = inside && (in_prefix || k1 - 1 <= i0 + off);
        full = inside && (in_prefix || k1 - 1 <= pos_lo);
        skip = p.causal && k0 > pos_lo + 31 && k0 >= prefix;
        if (p.docs != nullptr) {
            const int2 s = doc_span(ranges, k0, min(k1, p.sk));
            want = docs_meet(s, wg_span);
            whole = whole && docs_same(s, wg_span);
            full = full && docs_same(s, span);
            skip = skip || !docs_meet(s, span);
        }
    };

    // Up to four float outputs a row, as a regression has them, would leave most of a matrix instruction's 32 columns empty, each
    // of them as dear as a column of the scores' product: their sums are made by vector instructions, each half of the
    // lanes for its keys, in the first four registers of o (1e5 rows of 28 features, 2000 keys, 4 outputs: 326 us without this, 267 with it).
    const bool few = sizeof(T) == 4 && DP <= 64 && p.dv_d <= 4;     // (wider heads have no registers to spare)
    fx16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) o[db] = fx16{};
    float m = -kInf, l = 0.f;                                      // m in units of log 2

    int place_id = -1, next_id = -1;                               // id of key k0 + lane, one tile ahead
    const auto id_at = [&](int t) {
        const int k = t * TK + lane;
        return lane < TK && k < p.sk ? ids[k] : -1;
    };
    int buf = 0, tile = walk.next(look);
    bool whole = walk.is_whole, full = walk.is_full, skip = walk.is_skip;
    if (tile >= 0) {
        feed_k.issue(lds, tile * TK, min(TK, p.sk - tile * TK));
        feed_v.issue(lds + kTileBytes, tile * TK, min(TK, p.sk - tile * TK));
        if (p.docs != nullptr) next_id = id_at(tile);
    }
    while (tile >= 0) {
        const int k0 = tile * TK;
        char *lds_k = lds + buf * 2 * kTileBytes, *lds_v = lds_k + kTileBytes;
        const int next = walk.next(look);
        FD::wait();
        place_id = next_id;
        __syncthreads();                                           // this tile is there, the one before has been read
        buf ^= 1;
        if (next >= 0) {
            feed_k.issue(lds + buf * 2 * kTileBytes, next * TK, min(TK, p.sk - next * TK));
            feed_v.issue(lds + buf * 2 * kTileBytes + kTileBytes, next * TK, min(TK, p.sk - next * TK));
            if (p.docs != nullptr) next_id = id_at(next);
        }
        bool careful = false;
        if (!whole) {
            if (FD::nonfinite(lds_v)) lds_bad = tile;
            __syncthreads();
            careful = lds_bad == tile;
            if (careful) {                                         // clear them for the product, and add what they do to it below
                FD::clean_share(lds_v);
                __syncthreads();
            }
        }
        if (!skip) {
            fx16 s[KB];
#pragma unroll
            for (int kb = 0; kb < KB; kb++) s[kb] = fx16{};
            {   // fragments of the keys, read up to eight ahead of their products
                constexpr int n = KB * C, W = n < 8 ? n : 8;
                frag kf[W];
#pragma unroll
                for (int i = 0; i < W; i++) kf[i] = TL::rows(lds_k, at_lane, 32 * (i % KB), i / KB);
                FLK_KEEP_ORDER();
#pragma unroll
                for (int i = 0; i < n; i++) {
                    s[i % KB] = AT::mma(kf[i % W], qf[i / KB], s[i % KB]);
                    if (i + W < n) kf[i % W] = TL::rows(lds_k, at_lane, 32 * ((i + W) % KB), (i + W) / KB);
                    FLK_KEEP_ORDER();
                }
            }
            if constexpr (!kLate) {
                const float at = (float)(pos - k0 - 4 * half);
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        float grad;
                        s[kb][r] = score(s[kb][r], at - (float)(32 * kb + 8 * (r >> 2) + (r & 3)), grad);
                    }
            }
            Seen seen = {{~0u, ~0u}};
            if (!full) {
                uint64_t see = low_bits(last + 1 - k0);
                if (p.docs != nullptr) see &= same_id(place_id, id);
                seen = seen_from(see);
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int r = 0; r < 16; r++) s[kb][r] = seen.or_inf(s[kb][r], kb, r);
            }
            float top = -kInf;
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++) top = fmaxf(top, s[kb][r]);
            top = fmaxf(top, other_half(top));
            if constexpr (kLate) { float grad; top = score(top, 0.f, grad); }
            if (__any(top > m + (m == -kInf ? 0.f : kSlack))) {
                const float next_m = fmaxf(m, top);
                const float a = m == -kInf ? 0.f : __builtin_amdgcn_exp2f(m - next_m);
                l *= a;
                m = next_m;
#pragma unroll
                for (int db = 0; db < DB; db++) o[db] *= a;
            }
            const float base_m = m == -kInf ? 0.f : m - kLift<T>;
            // Weights and their product with the values.  The first fragments of the values are on their way before the first
            // weights are formed; the weights of the next 32 keys are formed between the products of the present ones.
            float sum[4] = {0.f, 0.f, 0.f, 0.f};                   // short chains: long ones would cost float data digits
            const auto weight = [&](int kb, int r) {
                float e;
                if constexpr (MOD == kPlain) e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], score.unit, -base_m));
                else if constexpr (!kLate) e = __builtin_amdgcn_exp2f(s[kb][r] - base_m);
                else {
                    e = __builtin_amdgcn_exp2f(__builtin_fmaf(score.r(s[kb][r]), -2.f * score.out, score.out - base_m));
                    e = seen.or_zero(e, kb, r);            // (a score of -inf may be seen: the cap makes it finite)
                }
                s[kb][r] = e;
                sum[r & 3] += e;
            };
            if (few) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    weight(0, r);
                    const fx4 v = *(const fx4 *)(lds_v + TL::at(8 * (r >> 2) + 4 * half + (r & 3), 0));
#pragma unroll
                    for (int c = 0; c < 4; c++) o[0][c] = __builtin_fmaf(s[0][r], v[c], o[0][c]);
                }
            } else {
                constexpr int F = ST * DB, EX = (16 + F - 1) / F;
                frag vf[F], pf[ST];
#pragma unroll
                for (int i = 0; i < F; i++) vf[i] = TL::cols(lds_v, at_lane, AT::KS * (i / DB), i % DB);
                FLK_KEEP_ORDER();
#pragma unroll
                for (int r = 0; r < 16; r++) weight(0, r);
#pragma unroll
                for (int kb = 0; kb < KB; kb++) {
#pragma unroll
                    for (int st = 0; st < ST; st++) pf[st] = pack<T>(s[kb], st);
                    FLK_KEEP_ORDER();
#pragma unroll
                    for (int i = 0; i < F; i++) {
                        o[i % DB] = AT::mma(vf[i], pf[i / DB], o[i % DB]);
                        if (kb + 1 < KB) {
                            vf[i] = TL::cols(lds_v, at_lane, 32 * (kb + 1) + AT::KS * (i / DB), i % DB);
#pragma unroll
                            for (int r = i * EX; r < (i + 1) * EX; r++)
                                if (r < 16) weight(kb + 1, r);
                        }
                        FLK_KEEP_ORDER();
                    }
                }
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (careful) {
                fx16 x[DB];
#pragma unroll
                for (int db = 0; db < DB; db++) x[db] = o[db];
                spread_nonfinite<T, TK, DB>(feed_v.base + k0 * feed_v.stride, feed_v.stride, p.sk - k0, p.dv_d, seen, 1.f, x);
#pragma unroll
                for (int db = 0; db < DB; db++) o[db] = x[db];
            }
        }
        tile = next;
        whole = walk.is_whole;
        full = walk.is_full;
        skip = walk.is_skip;
    }
    l += other_half(l);
    constexpr float kUnlift = 1.f / (1 << (int)kLift<T>);          // (exact, and the logarithm is as exact as without)
    if (few) {
#pragma unroll
        for (int c = 0; c < 4; c++) o[0][c] += other_half(o[0][c]);
    }
    if (p.parts > 1) {                                             // joined by attention_parts_kernel
        const int64_t rows_all = (int64_t)p.b * p.sq * p.hq, first = ((int64_t)b * p.sq + i0 + wave * 32) * p.hq + h;
        __syncthreads();
        store_rows<float, DP>(lds + wave * 32 * Tile<float, DP>::RB, [&](int db, int r) { return o[db][r] * kUnlift; },
                              p.part_o + (part * rows_all + first) * p.dv_d, (int64_t)p.hq * p.dv_d, p.sq - (i0 + wave * 32), p.dv_d, p.dv_d % 4 == 0);
        if (live && half == 0) {
            float *ml = p.part_ml + (part * rows_all + first + (int64_t)lane * p.hq) * 2;
            ml[0] = m;
            ml[1] = l * kUnlift;
        }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;                    // a row that sees nothing is zero
#pragma unroll
    for (int db = 0; db < DB; db++) o[db] *= inv;
    const int64_t row_o = (int64_t)p.hq * p.dv_d, at = (((int64_t)b * p.sq + i0 + wave * 32) * p.hq + h) * p.dv_d;
    const int rows = p.sq - (i0 + wave * 32);
    __syncthreads();
    char *mine = lds + wave * 32 * TL::RB;
    store_rows<T, DP>(mine, [&](int db, int r) { return o[db][r]; }, (T *)p.o + at, row_o, rows, p.dv_d, p.vec_v);
    if (p.rest != nullptr)
        store_rows<T, DP>(mine, [&](int db, int r) { return o[db][r] - (float)(T)o[db][r]; }, (T *)p.rest + at, row_o, rows, p.dv_d, p.vec_v);
    if (!live) return;
    if (half == 0 && p.lse != nullptr)
        p.lse[((int64_t)b * p.hq + h) * p.sq + row] = l == 0.f ? -kInf : m * kLn2 + __logf(l * kUnlift);
}

template <typename T> int launch_attention_fwd(const AttnArgs &a, int dp, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.b * a.hq * ((a.sq + kAttnRows - 1) / kAttnRows) * a.parts));
    FLK_ATTN_LAUNCH(attention_fwd_kernel, grid)
    return FLK_OK;
}
template int launch_attention_fwd<attn_t>(const AttnArgs &, int, hipStream_t);

}  // namespace flk
