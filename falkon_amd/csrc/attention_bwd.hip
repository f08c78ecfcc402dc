// Attention, backward (gfx950).  Compiled once per element type.
//
//   P_ij = exp(x_ij - lse_i),  dP_ij = dout_i.v_j,  delta_i = dout_i.out_i
//   dS_ij = P_ij (dP_ij - delta_i)                              (gradient of x)
//   dslope_h = -sum_ij dS_ij |pos_i - j|;   with a cap, dS <- dS (1 - tanh^2) before the products
//   dq_i = scale sum_j dS_ij k_j,   dk_j = scale sum_i dS_ij q_i,   dv_j = sum_i P_ij dout_i
//
// Two kernels instead of one with atomic sums of dq: seven products instead of five, and gradients that are the same run to
// run.  The first owns queries (dq, the rows' statistics, the slopes' partial sums), the second keys (dk, dv; it walks over
// the query heads that share its key head, so those are summed in registers).
//
// Infinities and NaNs reach what sees them as in these formulas, in tiles with a mask and without: a matrix product would carry them to
// what does not, so they never enter one whose other operand has hidden places.
#include "attention_common.h"

namespace flk {

template <typename T, int DP, int MOD>
__global__ void __launch_bounds__(kAttnThreads, sizeof(T) == 4 && DP > 64 ? 1 : 2) attention_dq_kernel(AttnArgs p) {
    typedef AttnType<T> AT;
    typedef typename AT::frag frag;
    typedef Tile<T, DP> TL;
    constexpr int TK = AT::kTile, KB = TK / 32, C = DP / AT::KS, DB = DP / 32, ST = 32 / AT::KS;
    typedef Feed<T, DP, TK> FD;
    constexpr int kTileBytes = TK * TL::RB;
    __shared__ __align__(16) char lds[4 * kTileBytes];
    __shared__ int lds_doc[8];
    __shared__ float lds_sum[4];
    __shared__ float lds_lse[kNarrow<T> ? kAttnThreads : 1];
    __shared__ int lds_bad;
    __shared__ Spoilt<DP> lds_spoilt[kAttnRows];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int heads = p.b * p.hq, pairs = p.b * p.hk;
    const int hb = blockIdx.x % heads, tiles_q = (p.sq + kAttnRows - 1) / kAttnRows;
    const int tile_q = tiles_q - 1 - blockIdx.x / heads % tiles_q, part = blockIdx.x / heads / tiles_q;
    const int b = hb % pairs / p.hk, hk = hb % p.hk, h = hk * p.group + hb / pairs;
    const int off = p.sk - p.sq;
    const int i0 = tile_q * kAttnRows, row = i0 + wave * 32 + (lane & 31);
    const bool live = row < p.sq;
    const int pos = row + off, pos_lo = i0 + wave * 32 + off;
    const int pos_end = min(i0 + kAttnRows, p.sq) + off;
    const Score<T, MOD> score(p.scale, p.cap, (MOD & kDecay) && p.slopes != nullptr ? p.slopes[h] : 0.f);
    const int prefix = p.prefix != nullptr ? max(min(p.prefix[b], p.sk), 0) : 0;
    const int last = p.causal ? min(max(pos, prefix - 1), p.sk - 1) : p.sk - 1;

    typename TL::Lane at_lane;
    at_lane.init();
    FD feed_k, feed_v;
    feed_k.init((const T *)p.k + b * p.ks.b + hk * p.ks.h, p.ks.s, p.d, p.vec);
    feed_v.init((const T *)p.v + b * p.vs.b + hk * p.vs.h, p.vs.s, p.dv_d, p.vec_v);
    const T *qrow = (const T *)p.q + b * p.qs.b + h * p.qs.h + (int64_t)row * p.qs.s;
    const T *grow = (const T *)p.dout + b * p.dos.b + h * p.dos.h + (int64_t)row * p.dos.s;
    const int64_t at = (((int64_t)b * p.sq + row) * p.hq + h) * p.dv_d;
    frag qf[C], gf[C];
    float delta = 0.f, size = 0.f;                                 // size: squared norm of dout
    unsigned bits = 0;
#pragma unroll
    for (int c = 0; c < C; c++) {
        union { ux4 u; frag f; } x, g, o, e;
        x.u = load_chunk<T>(qrow, 2 * c + half, p.d, live, p.vec);
        g.u = load_chunk<T>(grow, 2 * c + half, p.dv_d, live, p.vec_v);
        o.u = load_chunk<T>((const T *)p.out + at, 2 * c + half, p.dv_d, live, p.vec_v);
        e.u = load_chunk<T>((const T *)p.rest + at, 2 * c + half, p.dv_d, live && p.rest != nullptr, p.vec_v);
        qf[c] = x.f;
        gf[c] = g.f;
        bits |= bad_bits<T>(x.u) | bad_bits<T>(g.u);
#pragma unroll
        for (int i = 0; i < AT::E; i++) {
            delta += (float)g.f[i] * ((float)o.f[i] + (float)e.f[i]);
            if constexpr (kNarrow<T>) size += (float)g.f[i] * (float)g.f[i];
        }
    }
    delta += other_half(delta);
    // the statistics of this tile's rows, for both kernels; a row that sees nothing, or is none, has every p zero
    float lse = kInf;
    if (live) {
        const float x = p.lse[((int64_t)b * p.hq + h) * p.sq + row];
        lse = x == -kInf ? kInf : x * kScoreUnit;
    }
    bool bad_row = any_bad<T>(bits);
    bad_row |= __shfl_xor((int)bad_row, 32, 64) != 0;
    if (half == 0 && part == 0) {
        float *st = p.stats + ((int64_t)b * p.hq + h) * 3 * p.sq_pad + row;
        st[0] = bad_row ? kInf : lse;
        st[p.sq_pad] = delta;
        st[2 * p.sq_pad] = lse;
    }
    if constexpr (kNarrow<T>) {                                    // of rows that are finite and see something
        size += other_half(size);
        const bool counts = lse != kInf && !bad_row && __builtin_fabsf(delta) < kInf;
        float2 top = {__builtin_sqrtf(wave_maxf(counts ? size : 0.f)), wave_maxf(counts ? __builtin_fabsf(delta) : 0.f)};
        if (__any(bad_row)) top.x = -top.x;                        // (so that the other kernel has one thing to ask for; -0 too)
        if (lane == 0 && part == 0) p.sizes[(((int64_t)b * p.hq + h) * p.sq_pad + i0) / 32 + wave] = top;
    }
    const int bad_wave = (__any(bad_row) ? 1 : 0) | (__any(bad_row && lse != kInf) ? 2 : 0);
    if (lane == 0 && part == 0) p.bad_rows[(((int64_t)b * p.hq + h) * p.sq_pad + i0) / 32 + wave] = (unsigned char)bad_wave;
    if (p.dq == nullptr && p.dslopes_part == nullptr) return;      // only dk and dv are wanted

    int id = 0;
    int2 span = {0, 0}, wg_span = {0, 0};
    const int2 *ranges = p.doc_range + (int64_t)b * p.doc_blocks;
    const int *ids = p.doc_ids + (int64_t)b * p.doc_blocks * kDocBlock;
    if (threadIdx.x == 0) lds_bad = 0;
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

    fx16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) acc[db] = fx16{};
    // float16: the scores' gradients of a row (and its sums) are held times 2^lift.  The shift is a part of lse; it begins so high that
    // nothing is lost and falls where a tile would exceed 2^15 (as a running maximum does; then to 2^7, so that it seldom falls again).
    // (What remains of lse is small then and has all its digits: the slopes' gradient, in float, would show less.)
    constexpr float kFirstLift = kNarrow<T> ? 40.f : 0.f;
    float lift = kFirstLift, lse_lift = lse - kFirstLift;
    if constexpr (kNarrow<T>) lds_lse[threadIdx.x] = lse;
    // sum_j dS |dist|, sum_j dS and sum_j P |dist|: the second is what the rounding of out left in delta, and is taken out
    float far = 0.f, left = 0.f, reach = 0.f;

    int place_id = -1, next_id = -1;                               // id of key k0 + lane, one tile ahead
    const auto id_at = [&](int t) {
        const int k = t * TK + lane;
        return lane < TK && k < p.sk ? ids[k] : -1;
    };
    bool whole, full, skip;
    // A tile's part of the sums.  `careful`: its keys' infinities and NaNs are set to zero between the scores, which are formed from
    // them as they are, and the product with the scores' gradients.
    const auto visit = [&](int k0, char *lds_k, const char *lds_v, auto careful) __attribute__((always_inline)) {
        Seen seen = {{~0u, ~0u}};
        if (!full) {
            uint64_t see = low_bits(last + 1 - k0);
            if (p.docs != nullptr) see &= same_id(place_id, id);
            seen = seen_from(see);
        }
        const float at_key = (float)(pos - k0 - 4 * half);
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
            fx16 s = {}, dp = {};
            {   // fragments of keys and values, read up to four steps ahead of their products
                constexpr int W = C < 4 ? C : sizeof(T) == 2 && DP > 96 ? 2 : 4;     // (as the registers allow)
                frag kf[W], vf[W];
#pragma unroll
                for (int i = 0; i < W; i++) { kf[i] = TL::rows(lds_k, at_lane, 32 * kb, i); vf[i] = TL::rows(lds_v, at_lane, 32 * kb, i); }
                FLK_KEEP_ORDER();
#pragma unroll
                for (int c = 0; c < C; c++) {
                    s = AT::mma(kf[c % W], qf[c], s);
                    dp = AT::mma(vf[c % W], gf[c], dp);
                    if (c + W < C) { kf[c % W] = TL::rows(lds_k, at_lane, 32 * kb, c + W); vf[c % W] = TL::rows(lds_v, at_lane, 32 * kb, c + W); }
                    FLK_KEEP_ORDER();
                }
            }
            if constexpr (decltype(careful)::value) {
                if (!whole) FD::clean_block(lds_k, kb);
            }
            constexpr int F = ST * DB, WF = F < 4 ? F : 4;
            frag kt[WF], ds;
#pragma unroll
            for (int i = 0; i < WF; i++) kt[i] = TL::cols(lds_k, at_lane, 32 * kb + AT::KS * (i / DB), i % DB);
            FLK_KEEP_ORDER();
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float e, g, grad = 1.f;
                const float dist = at_key - (float)(32 * kb + 8 * (r >> 2) + (r & 3));
                if constexpr (MOD == kPlain) e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], score.unit, -lse_lift));
                else e = __builtin_amdgcn_exp2f(score(s[r], dist, grad) - lse_lift);
                g = e * (dp[r] - delta);
                if (!full) g = seen.or_zero(g, kb, r);
                if constexpr ((MOD & kDecay) != 0 && !decltype(careful)::value) {
                    if (p.dslopes_part != nullptr) {
                        if (!full) e = seen.or_zero(e, kb, r);
                        far += g * __builtin_fabsf(dist);
                        left += g;
                        reach += e * __builtin_fabsf(dist);
                    }
                }
                if constexpr ((MOD & kCap) != 0) g *= grad;
                s[r] = g;
            }
            if constexpr (kNarrow<T>) {
                float top = 0.f;
#pragma unroll
                for (int r = 0; r < 16; r++) top = fmaxf(top, __builtin_fabsf(s[r]));
                if (__any(top > 32768.f)) {
                    top = fmaxf(top, other_half(top));
                    const float drop = top > 32768.f ? (float)(__builtin_amdgcn_frexp_expf(fminf(top, 1e38f)) - 7) : 0.f;
                    const float by = __builtin_amdgcn_exp2f(-drop);
                    lift -= drop;
                    lse_lift = lds_lse[threadIdx.x] - lift;
                    if constexpr (!decltype(careful)::value) { far *= by; left *= by; reach *= by; }
#pragma unroll
                    for (int r = 0; r < 16; r++) s[r] *= by;
#pragma unroll
                    for (int db = 0; db < DB; db++) acc[db] *= by;
                }
            }
            FLK_KEEP_ORDER();
#pragma unroll
            for (int i = 0; i < F; i++) {
                if (i % DB == 0) ds = pack<T>(s, i / DB);
                acc[i % DB] = AT::mma(kt[i % WF], ds, acc[i % DB]);
                if (i + WF < F) kt[i % WF] = TL::cols(lds_k, at_lane, 32 * kb + AT::KS * ((i + WF) / DB), (i + WF) % DB);
                FLK_KEEP_ORDER();
            }
        }
        if constexpr (decltype(careful)::value) {
            // (a score's gradient is zero, because its weight or the cap's derivative is, or NaN where its key is not finite)
            if (!whole) lds_spoilt[wave * 32 + (lane & 31)].note(feed_k.base + k0 * feed_k.stride, feed_k.stride, min(TK, p.sk - k0), p.d, seen);
        }
    };
    int buf = 0, tile = walk.next(look);
    whole = walk.is_whole, full = walk.is_full, skip = walk.is_skip;
    bool bad = false;                                              // a key that is not finite, hidden from some row of the workgroup
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
        __syncthreads();
        buf ^= 1;
        if (next >= 0) {
            feed_k.issue(lds + buf * 2 * kTileBytes, next * TK, min(TK, p.sk - next * TK));
            feed_v.issue(lds + buf * 2 * kTileBytes + kTileBytes, next * TK, min(TK, p.sk - next * TK));
            if (p.docs != nullptr) next_id = id_at(next);
        }
        if (!whole) bad |= FD::nonfinite(lds_k);
        if (!skip) visit(k0, lds_k, lds_v, std::false_type{});
        tile = next;
        whole = walk.is_whole;
        full = walk.is_full;
        skip = walk.is_skip;
    }
    // Such keys' part of the last product reached rows that hide them: it is formed again from all tiles, one at a time.  (In a loop of
    // its own: a branch in the middle of the one above takes hundreds of its registers to memory.  The slopes' sums stand: they have no
    // product with the keys, and are masked.)
    if (bad) lds_bad = 1;
    __syncthreads();
    const float unlift = __builtin_amdgcn_exp2f(-lift);            // of the slopes' sums
    const bool again = p.dq != nullptr && lds_bad != 0;
    if (again) {
#pragma unroll
        for (int db = 0; db < DB; db++) acc[db] = fx16{};
        lift = kFirstLift;
        if constexpr (kNarrow<T>) lse_lift = lds_lse[threadIdx.x] - lift;
        lds_spoilt[wave * 32 + (lane & 31)].clear();
        walk.start((int)(tiles_k * part / p.parts), (int)(tiles_k * (part + 1) / p.parts));
        while ((tile = walk.next(look)) >= 0) {
            const int k0 = tile * TK, n = min(TK, p.sk - k0);
            __syncthreads();                                       // the tile before has been read
            feed_k.issue(lds, k0, n);
            feed_v.issue(lds + kTileBytes, k0, n);
            if (p.docs != nullptr) place_id = id_at(tile);
            whole = walk.is_whole;
            full = walk.is_full;
            FD::wait();
            __syncthreads();
            at_lane.renew();
            visit(k0, lds, lds + kTileBytes, std::true_type{});    // (a wave that sees nothing of it takes part in the barriers)
        }
    }
    if ((MOD & kDecay) != 0 && p.dslopes_part != nullptr) {                        // in a fixed order: lanes, then waves
        far += other_half(far);
        left += other_half(left);
        reach += other_half(reach);
        float x = live && half == 0 ? (left * (reach * unlift) - far) * unlift : 0.f;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
        if (lane == 0) lds_sum[wave] = x;
        __syncthreads();
        if (threadIdx.x == 0)
            p.dslopes_part[((int64_t)h * p.b + b) * tiles_q + tile_q] = (lds_sum[0] + lds_sum[1]) + (lds_sum[2] + lds_sum[3]);
    }
    if (p.dq == nullptr) return;
    __syncthreads();
    if (again) lds_spoilt[wave * 32 + (lane & 31)].mark(acc);
    const float unscale = p.scale * score.kGrad * __builtin_amdgcn_exp2f(-lift);
    const int64_t to = (((int64_t)b * p.sq + i0 + wave * 32) * p.hq + h) * p.d, row_q = (int64_t)p.hq * p.d;
    const auto value = [&](int db, int r) { return acc[db][r] * unscale; };
    const int rows = p.sq - (i0 + wave * 32);
    if (p.parts == 1) store_rows<T, DP>(lds + wave * 32 * TL::RB, value, (T *)p.dq + to, row_q, rows, p.d, p.vec);
    else                                                           // parts in float, added by attention_join_kernel
        store_rows<float, DP>(lds + wave * 32 * Tile<float, DP>::RB, value, p.dq_part + part * (int64_t)p.b * p.sq * row_q + to, row_q, rows, p.d, p.d % 4 == 0);
}

// Whether the dk / dv kernel's fragments and sums (keys, values, dk and dv of 32 keys in registers) leave room for one wave a SIMD only
template <typename T, int DP> constexpr bool kAlone = sizeof(T) == 4 ? DP >= 64 : DP > 64;

template <typename T, int DP, int MOD>
__global__ void __launch_bounds__(kAttnThreads, (kAlone<T, DP> ? 1 : 2)) attention_dkv_kernel(AttnArgs p) {
    typedef AttnType<T> AT;
    typedef typename AT::frag frag;
    typedef Tile<T, DP> TL;
    constexpr int TQ = AT::kTile, QB = TQ / 32, C = DP / AT::KS, DB = DP / 32, ST = 32 / AT::KS;
    typedef Feed<T, DP, TQ> FD;
    constexpr int kTileBytes = TQ * TL::RB;
    __shared__ __align__(16) char lds[4 * kTileBytes];
    __shared__ __align__(16) float lds_stat[2][2][TQ];             // lse and delta of a tile's rows
    __shared__ int lds_doc[8];
    __shared__ int lds_bad[4];
    __shared__ float lds_size[4][3];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int pairs = p.b * p.hk, tiles_k = (p.sk + kAttnRows - 1) / kAttnRows;
    const int splits = p.head_parts * p.row_parts, pair = blockIdx.x % pairs, split = blockIdx.x / pairs % splits;
    const int tile_k = blockIdx.x / pairs / splits, head_part = split % p.head_parts, row_part = split / p.head_parts;
    const int b = pair / p.hk, hk = pair % p.hk;
    const int off = p.sk - p.sq;
    const int k0 = tile_k * kAttnRows, k_lo = k0 + wave * 32, key = k_lo + (lane & 31);
    const bool live = key < p.sk;
    const int prefix = p.prefix != nullptr ? max(min(p.prefix[b], p.sk), 0) : 0;
    const int first = p.causal && key >= prefix ? key - off : 0;   // first row that sees this key

    // rows that may see a key of this tile: with the causal mask those at or behind its first key, or all for a prefix.
    // (A row past the last one is masked like a hidden one: zero times an infinity of a key would be its score.)
    const int lo = p.causal && k0 >= prefix ? max(k0 - off, 0) : 0;
    const int tile_lo = lo / TQ, tile_end = (p.sq + TQ - 1) / TQ;
    const int64_t tiles_q = max(0, tile_end - tile_lo);
    const int walk_lo = tile_lo + (int)(tiles_q * row_part / p.row_parts), walk_end = tile_lo + (int)(tiles_q * (row_part + 1) / p.row_parts);
    // the heads that share this key head, one after the other; the tiles to visit are the same for each
    int head = p.group * head_part / p.head_parts;                 // of the tile on its way
    const int head_end = p.group * (head_part + 1) / p.head_parts;
    // Whether any of the rows that this workgroup goes over is not finite.  (Asked for first, so that the answer is on its way together
    // with keys and values.)
    // float16: also the largest norm of a row of dout, and |delta|.
    bool bad = false;
    float dout_size = 0.f, delta_size = 0.f;
    const int64_t line0 = (int64_t)b * p.hq + hk * p.group + head;
    if constexpr (kNarrow<T>) {
        const int first_of = walk_lo * TQ / 32, n = walk_end * TQ / 32 - first_of, all = n * (head_end - head);
        for (int i = threadIdx.x; i < all; i += kAttnThreads) {
            const float2 x = p.sizes[(line0 + i / n) * (p.sq_pad / 32) + first_of + i % n];
            bad |= __builtin_signbitf(x.x);
            dout_size = fmaxf(dout_size, __builtin_fabsf(x.x));
            delta_size = fmaxf(delta_size, x.y);
        }
    } else {
        const int first_of = walk_lo * TQ / kAttnRows, n = (walk_end * TQ + kAttnRows - 1) / kAttnRows - first_of, all = n * (head_end - head);
        for (int i = threadIdx.x; i < all; i += kAttnThreads)
            bad |= ((const int *)p.bad_rows)[(line0 + i / n) * (p.sq_pad / kAttnRows) + first_of + i % n] != 0;
    }
    const T *krow = (const T *)p.k + b * p.ks.b + hk * p.ks.h + (int64_t)key * p.ks.s;
    const T *vrow = (const T *)p.v + b * p.vs.b + hk * p.vs.h + (int64_t)key * p.vs.s;
    typename TL::Lane at_lane;
    at_lane.init();
    frag kf[C], vf[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        union { ux4 u; frag f; } x, y;
        x.u = load_chunk<T>(krow, 2 * c + half, p.d, live, p.vec);
        y.u = load_chunk<T>(vrow, 2 * c + half, p.dv_d, live, p.vec_v);
        kf[c] = x.f;
        vf[c] = y.f;
    }
    int id = 0;
    int2 span = {0, 0}, wg_span = {0, 0};
    const int2 *ranges = p.doc_range + (int64_t)b * p.doc_blocks;
    const int *ids = p.doc_ids + (int64_t)b * p.doc_blocks * kDocBlock;
    const bool bad_wave = __any(bad);
    if (lane == 0) lds_bad[wave] = bad_wave;
    // float16: weights are held times 2^10, and the scores' gradients times 2^10 and a power of two, `fit`, that bounds them by 2^11:
    // |dP - delta| is at most the largest norm of a row of dout times that of a key's row of v, plus the largest |delta|.  (Five more
    // bits are left, since a weight exceeds one by the rounding of scores of millions.)
    constexpr float kLift = kNarrow<T> ? 10.f : 0.f;
    float fit = 1.f;
    if constexpr (kNarrow<T>) {
        float v_size = 0.f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < AT::E; i++) v_size += (float)vf[c][i] * (float)vf[c][i];
        v_size += other_half(v_size);
        v_size = v_size < kInf ? v_size : 0.f;
        dout_size = wave_maxf(dout_size);
        delta_size = wave_maxf(delta_size);
        v_size = wave_maxf(v_size);
        if (lane == 0) { lds_size[wave][0] = dout_size; lds_size[wave][1] = delta_size; lds_size[wave][2] = v_size; }
    }
    if (p.docs != nullptr) {
        const int raw = live ? ids[key] : -1;
        span = {wave_min(raw), wave_max(raw)};
        if (lane == 0) { lds_doc[wave] = span.x; lds_doc[4 + wave] = span.y; }
        id = raw;
    }
    __syncthreads();
    bad = (lds_bad[0] | lds_bad[1] | lds_bad[2] | lds_bad[3]) != 0;
    if constexpr (kNarrow<T>) {
        float x[3];
#pragma unroll
        for (int i = 0; i < 3; i++) x[i] = fmaxf(fmaxf(lds_size[0][i], lds_size[1][i]), fmaxf(lds_size[2][i], lds_size[3][i]));
        const float most = 1.01f * (x[0] * __builtin_sqrtf(x[2]) + x[1]);
        if (most > 0.f) fit = __builtin_amdgcn_exp2f((float)(1 - max(__builtin_amdgcn_frexp_expf(most), -100)));
    }
    if (p.docs != nullptr) {
        wg_span.x = min(min(lds_doc[0], lds_doc[1]), min(lds_doc[2], lds_doc[3]));
        wg_span.y = max(max(lds_doc[4], lds_doc[5]), max(lds_doc[6], lds_doc[7]));
    }
    const auto look = [&](int t, bool &want, bool &whole, bool &full, bool &skip) {
        const int i0 = t * TQ, i1 = min(i0 + TQ, p.sq);
        const bool inside = i0 + TQ <= p.sq;
        whole = inside && (!p.causal || k0 + kAttnRows - 1 <= i0 + off || k0 + kAttnRows <= prefix);
        full = inside && (!p.causal || k_lo + 31 <= i0 + off || k_lo + 32 <= prefix);
        skip = p.causal && k_lo > i0 + TQ - 1 + off && k_lo >= prefix;
        if (p.docs != nullptr) {
            const int2 s = doc_span(ranges, i0 + off, i1 + off);
            want = docs_meet(s, wg_span);
            whole = whole && docs_same(s, wg_span);
            full = full && docs_same(s, span);
            skip = skip || !docs_meet(s, span);
        }
    };

    fx16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) dk[db] = dv[db] = fx16{};

    Score<T, MOD> score(p.scale, p.cap, 0.f);
    FD feed_q, feed_g;
    feed_q.init((const T *)p.q + b * p.qs.b + (hk * p.group + head) * p.qs.h, p.qs.s, p.d, p.vec);
    feed_g.init((const T *)p.dout + b * p.dos.b + (hk * p.group + head) * p.dos.h, p.dos.s, p.dv_d, p.vec_v);
    const float *stats = p.stats + ((int64_t)b * p.hq + hk * p.group + head) * 3 * p.sq_pad;
    // a tile's statistics (padded to whole tiles of 128 rows) pass through registers of its first threads
    float r_lse = 0.f, r_delta = 0.f;
    int place_id = -1, next_id = -1;                               // id of row i0 + lane, one tile ahead
    const bool mine = (int)threadIdx.x < TQ;
    const auto issue = [&](int t, char *to) {
        const int i0 = t * TQ, rows = min(TQ, p.sq - i0);
        feed_q.issue(to, i0, rows);
        feed_g.issue(to + kTileBytes, i0, rows);
        if (mine) {
            r_lse = stats[i0 + threadIdx.x];
            r_delta = stats[p.sq_pad + i0 + threadIdx.x];
        }
        if (p.docs != nullptr) next_id = lane < rows ? ids[i0 + off + lane] : -1;
    };
    const auto put = [&](int to) {
        if (mine) { lds_stat[to][0][threadIdx.x] = r_lse - kLift; lds_stat[to][1][threadIdx.x] = r_delta * fit; }
    };
    TileWalk walk, again;
    walk.start(walk_lo, walk_end);
    int tile = walk.next(look);
    again = walk;                                                  // the first 64 tiles as they were found
    const int first_tile = tile;
    const bool first_whole = walk.is_whole, first_full = walk.is_full, first_skip = walk.is_skip;
    const auto advance = [&]() {
        const int t = walk.next(look);
        if (t >= 0 || head + 1 >= head_end) return t;
        head++;
        feed_q.base += p.qs.h;
        feed_g.base += p.dos.h;
        stats += 3 * p.sq_pad;
        walk = again;
        walk.is_whole = first_whole;
        walk.is_full = first_full;
        walk.is_skip = first_skip;
        return first_tile;
    };
    const auto decay = [&](int hg) {
        if constexpr ((MOD & kDecay) != 0) score.slope = p.slopes != nullptr ? p.slopes[hk * p.group + hg] * kScoreUnit : 0.f;
    };
    if (tile >= 0) {
        decay(head);
        int buf = 0, head_of = head;                               // head_of: of the tile in use
        bool whole = walk.is_whole, full = walk.is_full, skip = walk.is_skip;
        issue(tile, lds);
        put(0);
        while (tile >= 0) {
            const int i0 = tile * TQ;
            char *lds_q = lds + buf * 2 * kTileBytes, *lds_g = lds_q + kTileBytes;
            const float *lse_of = lds_stat[buf][0], *delta_of = lds_stat[buf][1];
            const int next = advance();
            FD::wait();
            place_id = next_id;
            __syncthreads();
            buf ^= 1;
            if (next >= 0) issue(next, lds + buf * 2 * kTileBytes);
            if (bad) {                                             // rows that are not finite, which attention_bad_rows_kernel adds
                FD::clean_share(lds_q);
                FD::clean_share(lds_g);
                __syncthreads();
            }
            if (!skip) {
                Seen seen = {{~0u, ~0u}};
                if (!full) {
                    uint64_t see = low_bits(p.sq - i0) & ~low_bits(first - i0);
                    if (p.docs != nullptr) see &= same_id(place_id, id);
                    seen = seen_from(see);
                }
                const float at_row = (float)(i0 + off + 4 * half - key);
                at_lane.renew();
                constexpr int kAhead = kAlone<T, DP> ? 4 : 2;         // steps that fragments are read ahead
                constexpr int N = QB * C, W = N < kAhead ? N : kAhead, F = ST * DB, NF = QB * F, WF = NF < kAhead ? NF : kAhead;
                frag qf[W], gf[W], gt[WF], qt[WF], pf[QB][ST], sf[QB][ST];    // pf, sf: weights and their gradients, rounded
                fx16 s[QB], dp[QB];
                fx4 lse[2], delta[2];                              // of four registers' rows, one group ahead
                const auto read_rows = [&](int n) {
                    qf[n % W] = TL::rows(lds_q, at_lane, 32 * (n / C), n % C);
                    gf[n % W] = TL::rows(lds_g, at_lane, 32 * (n / C), n % C);
                };
                const auto read_cols = [&](int n) {
                    const int row = 32 * (n / F) + AT::KS * (n % F / DB);
                    gt[n % WF] = TL::cols(lds_g, at_lane, row, n % DB);
                    qt[n % WF] = TL::cols(lds_q, at_lane, row, n % DB);
                };
                const auto read_stats = [&](int qb, int g4) {
                    lse[g4 & 1] = *(const fx4 *)(lse_of + 32 * qb + 8 * g4 + 4 * half);
                    delta[g4 & 1] = *(const fx4 *)(delta_of + 32 * qb + 8 * g4 + 4 * half);
                };
                const auto scores = [&](int n) {                   // one step of the products behind scores and their gradients
                    const int qb = n / C, c = n % C;
                    s[qb] = AT::mma(qf[n % W], kf[c], c == 0 ? fx16{} : s[qb]);
                    dp[qb] = AT::mma(gf[n % W], vf[c], c == 0 ? fx16{} : dp[qb]);
                    if (n + W < N) read_rows(n + W);
                };
                // the weights of two registers, rounded at once so that they take a quarter of the registers
                const auto weights = [&](int qb, int pair, bool masked) {
                    typedef T two __attribute__((ext_vector_type(2)));
                    if (pair % 2 == 0 && pair < 6) read_stats(qb, pair / 2 + 1);
                    float e[2], g[2];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int r = 2 * pair + k;
                        const float li = lse[r >> 2 & 1][r & 3], de = delta[r >> 2 & 1][r & 3];
                        float grad = 1.f;
                        if constexpr (MOD == kPlain) e[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qb][r], score.unit, -li));
                        else e[k] = __builtin_amdgcn_exp2f(score(s[qb][r], at_row + (float)(32 * qb + 8 * (r >> 2) + (r & 3)), grad) - li);
                        float x = kNarrow<T> ? __builtin_fmaf(dp[qb][r], fit, -de) : dp[qb][r] - de;
                        if constexpr ((MOD & kCap) != 0) x *= grad;
                        if (masked) e[k] = seen.or_zero(e[k], qb, r);
                        g[k] = times_or_zero(e[k], x);                       // a hidden place stays zero whatever x is
                    }
                    union { frag f; two t[AT::E / 2]; } u, v;
                    const int st = 2 * pair / AT::E, at2 = pair % (AT::E / 2);
                    u.f = pf[qb][st];
                    v.f = sf[qb][st];
                    u.t[at2] = two{(T)e[0], (T)e[1]};
                    v.t[at2] = two{(T)g[0], (T)g[1]};
                    pf[qb][st] = u.f;
                    sf[qb][st] = v.f;
                };
                const auto gradients = [&](int n) {                // one step of the gradients' products
                    const int qb = n / F, i = n % F;
                    dv[i % DB] = AT::mma(gt[n % WF], pf[qb][i / DB], dv[i % DB]);
                    dk[i % DB] = AT::mma(qt[n % WF], sf[qb][i / DB], dk[i % DB]);
                    if (n + WF < NF) read_cols(n + WF);
                };
#pragma unroll
                for (int n = 0; n < W; n++) read_rows(n);
                FLK_KEEP_ORDER();
                if constexpr (kAlone<T, DP> && QB == 2) {
                    // One wave a SIMD has to keep its matrix cores busy by itself: the weights of the first 32 rows are formed
                    // between the score products of the second, and theirs between the gradient products of the first.  No
                    // branch may stand between them, so every tile is masked (2 x 4096 positions, 32 heads of 128, causal: the whole
                    // backward pass 1.37 ms with the steps one after the other, 1.23 ms so).
                    constexpr int EC = (8 + C - 1) / C, EF = (8 + F - 1) / F;   // pairs a step
#pragma unroll
                    for (int c = 0; c < C; c++) { scores(c); FLK_KEEP_ORDER(); }
                    read_stats(0, 0);
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        scores(C + c);
#pragma unroll
                        for (int n = c * WF / C; n < (c + 1) * WF / C; n++) read_cols(n);
#pragma unroll
                        for (int r = c * EC; r < (c + 1) * EC; r++)
                            if (r < 8) weights(0, r, true);
                        FLK_KEEP_ORDER();
                    }
                    read_stats(1, 0);
#pragma unroll
                    for (int i = 0; i < F; i++) {
                        gradients(i);
#pragma unroll
                        for (int r = i * EF; r < (i + 1) * EF; r++)
                            if (r < 8) weights(1, r, true);
                        FLK_KEEP_ORDER();
                    }
#pragma unroll
                    for (int i = F; i < NF; i++) { gradients(i); FLK_KEEP_ORDER(); }
                } else {
                    const bool masked = !(whole && full);
#pragma unroll
                    for (int qb = 0; qb < QB; qb++) {
#pragma unroll
                        for (int c = 0; c < C; c++) { scores(qb * C + c); FLK_KEEP_ORDER(); }
                        if (qb == 0) {
#pragma unroll
                            for (int n = 0; n < WF; n++) read_cols(n);
                        }
                        read_stats(qb, 0);
                        FLK_KEEP_ORDER();
#pragma unroll
                        for (int r = 0; r < 8; r++) weights(qb, r, masked);
                        FLK_KEEP_ORDER();
#pragma unroll
                        for (int i = 0; i < F; i++) { gradients(qb * F + i); FLK_KEEP_ORDER(); }
                    }
                }
            }
            if (next >= 0) put(buf);
            if (head != head_of) { head_of = head; decay(head); }
            tile = next;
            whole = walk.is_whole;
            full = walk.is_full;
            skip = walk.is_skip;
        }
    }
    __syncthreads();
    const float lowered = __builtin_amdgcn_exp2f(-kLift), unscale = p.scale * Score<T, MOD>::kGrad * lowered / fit;
    const int rows = p.sk - k_lo;
    const int64_t line = (int64_t)b * p.sk + k_lo, at_k = (line * p.hk + hk) * p.d, at_v = (line * p.hk + hk) * p.dv_d;
    const int64_t row_k = (int64_t)p.hk * p.d, row_v = (int64_t)p.hk * p.dv_d;
    if (splits == 1) {
        char *mine = lds + wave * 32 * TL::RB;
        store_rows<T, DP>(mine, [&](int db, int r) { return dk[db][r] * unscale; }, (T *)p.dk + at_k, row_k, rows, p.d, p.vec);
        store_rows<T, DP>(mine, [&](int db, int r) { return dv[db][r] * lowered; }, (T *)p.dv + at_v, row_v, rows, p.dv_d, p.vec_v);
    } else {                                                       // parts in float, added by attention_join_kernel
        const int64_t nk = (int64_t)p.b * p.sk * row_k, nv = (int64_t)p.b * p.sk * row_v;
        char *mine = lds + wave * 32 * Tile<float, DP>::RB;
        store_rows<float, DP>(mine, [&](int db, int r) { return dk[db][r] * unscale; }, p.dkv_part + split * nk + at_k, row_k, rows, p.d, p.d % 4 == 0);
        store_rows<float, DP>(mine, [&](int db, int r) { return dv[db][r] * lowered; }, p.dkv_part + splits * nk + split * nv + at_v, row_v, rows, p.dv_d,
                              p.d % 4 == 0 && p.dv_d % 4 == 0);
    }
}

// What rows of q and dout with infinities or NaNs, which have no weight in the kernel above, do to dk and dv of the keys that see
// them: one row after the other, by vector instructions, added to what was written (to the first of its parts).  A product of matrices
// would carry their NaNs (zero times an infinity) to the keys that do not see them.  A workgroup goes over the rows for 128 keys, and has
// nothing to do where all rows are finite (4 to 5 us; as a branch of the kernel above it took 5 % of its time by its registers).
template <typename T, int DP, int MOD>
__global__ void __launch_bounds__(kAttnThreads) attention_bad_rows_kernel(AttnArgs p) {
    typedef AttnType<T> AT;
    typedef typename AT::frag frag;
    constexpr int C = DP / AT::KS, DB = DP / 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int pairs = p.b * p.hk, pair = blockIdx.x % pairs, tile_k = blockIdx.x / pairs, b = pair / p.hk, hk = pair % p.hk;
    const int off = p.sk - p.sq, k_lo = tile_k * kAttnRows + wave * 32, key = k_lo + (lane & 31);
    const bool live = key < p.sk;
    const int64_t flags = p.sq_pad / 32, line0 = (int64_t)b * p.hq + hk * p.group;
    // (a key head's flags lie one after the other)
    bool bad = false;
    for (int64_t i = lane; i < flags * p.group / 4; i += 64) bad |= (((const int *)p.bad_rows)[line0 * flags / 4 + i] & 0x02020202) != 0;
    if (!__any(bad)) return;
    const int prefix = p.prefix != nullptr ? max(min(p.prefix[b], p.sk), 0) : 0;
    const int first = p.causal && key >= prefix ? key - off : 0;   // first row that sees this key
    const int *ids = p.doc_ids + (int64_t)b * p.doc_blocks * kDocBlock;
    const int id = p.docs != nullptr && live ? ids[key] : 0;
    const T *krow = (const T *)p.k + b * p.ks.b + hk * p.ks.h + (int64_t)key * p.ks.s;
    const T *vrow = (const T *)p.v + b * p.vs.b + hk * p.vs.h + (int64_t)key * p.vs.s;
    frag kf[C], vf[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        union { ux4 u; frag f; } x, y;
        x.u = load_chunk<T>(krow, 2 * c + half, p.d, live, p.vec);
        y.u = load_chunk<T>(vrow, 2 * c + half, p.dv_d, live, p.vec_v);
        kf[c] = x.f;
        vf[c] = y.f;
    }
    fx16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) dk[db] = dv[db] = fx16{};
    bool all_nan = false;
    for (int g = 0; g < p.group; g++) {
        const int h = hk * p.group + g;
        const T *q0 = (const T *)p.q + b * p.qs.b + h * p.qs.h;
        const T *g0 = (const T *)p.dout + b * p.dos.b + h * p.dos.h;
        const Score<T, MOD> score(p.scale, p.cap, (MOD & kDecay) && p.slopes != nullptr ? p.slopes[h] : 0.f);
        const float *lse_of = p.stats + (line0 + g) * 3 * p.sq_pad, *delta_of = lse_of + p.sq_pad, *true_lse_of = delta_of + p.sq_pad;
        uint64_t todo = 0;
        int i0 = (p.causal && k_lo >= prefix ? max(k_lo - off, 0) : 0) / 32 * 32 - 32;
#pragma unroll 1
        while (!all_nan) {                                         // (which is what they soon are where no row is finite)
            while (todo == 0 && (i0 += 32) < p.sq) {
                if (!(p.bad_rows[(line0 + g) * flags + i0 / 32] & 2)) continue;
                const int at = i0 + (lane & 31);
                todo = (uint32_t)__ballot(lse_of[at] == kInf && true_lse_of[at] != kInf);
            }
            if (todo == 0) break;
            const int i = i0 + __builtin_ctzll(todo);
            todo &= todo - 1;
            const float lse = true_lse_of[i], delta = delta_of[i];
            const bool see = live && i >= first && (p.docs == nullptr || (id >= 0 && ids[i + off] == id));
            if (!__any(see)) continue;
            const T *qi = q0 + i * p.qs.s, *gi = g0 + i * p.dos.s;
            float s = 0.f, dp = 0.f, grad = 1.f;
#pragma unroll
            for (int c = 0; c < C; c++) {
                union { ux4 u; frag f; } x, y;
                x.u = load_chunk<T>(qi, 2 * c + half, p.d, true, p.vec);
                y.u = load_chunk<T>(gi, 2 * c + half, p.dv_d, true, p.vec_v);
#pragma unroll
                for (int j = 0; j < AT::E; j++) { s += (float)x.f[j] * (float)kf[c][j]; dp += (float)y.f[j] * (float)vf[c][j]; }
            }
            s += other_half(s);
            dp += other_half(dp);
            const float e = __builtin_amdgcn_exp2f(score(s, (float)(i + off - key), grad) - lse);
            float x = dp - delta;
            if constexpr ((MOD & kCap) != 0) x *= grad;
            const float ds = times_or_zero(e, x);
            int c0 = 4 * half;
            asm volatile("" : "+v"(c0));                           // (or the comparisons below are made ahead and kept)
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int c = c0 + 32 * db + 8 * (r >> 2) + (r & 3);
                    const float qc = c < p.d ? (float)qi[c] : 0.f, gc = c < p.dv_d ? (float)gi[c] : 0.f;
                    if (see) {
                        dk[db][r] += ds * qc;
                        dv[db][r] += __builtin_fabsf(gc) < kInf ? e * gc : __builtin_nanf("");
                    }
                }
            bool nan = true;
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int c = c0 + 32 * db + 8 * (r >> 2) + (r & 3);
                    nan &= (c >= p.d || dk[db][r] != dk[db][r]) && (c >= p.dv_d || dv[db][r] != dv[db][r]);
                }
            all_nan = !__any(live && !nan);
        }
    }
    if (!live) return;
    const int splits = p.head_parts * p.row_parts;
    const int64_t keys = (int64_t)p.b * p.sk * p.hk, row = ((int64_t)b * p.sk + key) * p.hk + hk;
    const float unscale = p.scale * Score<T, MOD>::kGrad;
    const auto add = [&](auto *to, const fx16 *x, int n, float by) {
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = 32 * db + 8 * (r >> 2) + 4 * half + (r & 3);
                if (c < n) to[c] = (std::remove_reference_t<decltype(*to)>)((float)to[c] + x[db][r] * by);
            }
    };
    if (splits == 1) {
        add((T *)p.dk + row * p.d, dk, p.d, unscale);
        add((T *)p.dv + row * p.dv_d, dv, p.dv_d, 1.f);
    } else {
        add(p.dkv_part + row * p.d, dk, p.d, unscale);
        add(p.dkv_part + splits * keys * p.d + row * p.dv_d, dv, p.dv_d, 1.f);
    }
}

template <typename T> int launch_attention_dq(const AttnArgs &a, int dp, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.b * a.hq * ((a.sq + kAttnRows - 1) / kAttnRows) * a.parts));
    FLK_ATTN_LAUNCH(attention_dq_kernel, grid)
    return FLK_OK;
}
template <typename T> int launch_attention_dkv(const AttnArgs &a, int dp, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.b * a.hk * a.head_parts * a.row_parts * ((a.sk + kAttnRows - 1) / kAttnRows)));
    FLK_ATTN_LAUNCH(attention_dkv_kernel, grid)
    const dim3 tiles((unsigned)((int64_t)a.b * a.hk * ((a.sk + kAttnRows - 1) / kAttnRows)));
    if (a.sq > 0) FLK_ATTN_LAUNCH_KIND(attention_bad_rows_kernel, tiles)
    return FLK_OK;
}
template int launch_attention_dq<attn_t>(const AttnArgs &, int, hipStream_t);
template int launch_attention_dkv<attn_t>(const AttnArgs &, int, hipStream_t);

}  // namespace flk
