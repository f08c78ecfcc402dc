// Attention, backward (gfx950).  Compiled once per element type.
//
//   P_ij = exp(x_ij - lse_i),  dP_ij = dout_i.v_j,  delta_i = dout_i.out_i
//   dS_ij = P_ij (dP_ij - delta_i)                              (gradient of x)
//   dslope_h = -sum_ij dS_ij |pos_i - j|;   with a cap, dS <- dS (1 - tanh^2) before the products
//   dq_i = scale sum_j dS_ij k_j,   dk_j = scale sum_i dS_ij q_i,   dv_j = sum_i P_ij dout_i
//
// Two kernels instead of one with atomic sums of dq: seven products instead of five, and gradients that are the same run to
// run.  The first owns queries (dq, delta, the slopes' partial sums), the second keys (dk, dv; it walks over the query heads
// that share its key head, so those are summed in registers).
#include "attention_common.h"

namespace flk {

template <typename T, int DP, bool MOD>
__global__ void __launch_bounds__(kAttnThreads, 2) attention_dq_kernel(AttnArgs p) {
    typedef AttnType<T> AT;
    typedef typename AT::frag frag;
    typedef Tile<T, DP> TL;
    constexpr int TK = AT::kTile, KB = TK / 32, C = DP / AT::KS, DB = DP / 32, ST = 32 / AT::KS;
    __shared__ __align__(16) char lds_k[TK * TL::RB];
    __shared__ __align__(16) char lds_v[TK * TL::RB];
    __shared__ int lds_doc[8];
    __shared__ float lds_sum[4];
    __shared__ int lds_bad;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int heads = p.b * p.hq, pairs = p.b * p.hk;
    const int hb = blockIdx.x % heads, tiles_q = (p.sq + kAttnRows - 1) / kAttnRows;
    const int tile_q = tiles_q - 1 - blockIdx.x / heads;
    const int b = hb % pairs / p.hk, hk = hb % p.hk, h = hk * p.group + hb / pairs;
    const int off = p.sk - p.sq;
    const int i0 = tile_q * kAttnRows, row = i0 + wave * 32 + (lane & 31);
    const bool live = row < p.sq;
    const int pos = row + off;
    const int pos_lo = i0 + wave * 32 + off;
    const int pos_end = min(i0 + kAttnRows, p.sq) + off;
    const float slope = MOD && p.slopes != nullptr ? p.slopes[h] : 0.f;
    const int prefix = p.prefix != nullptr ? min(p.prefix[b], p.sk) : 0;

    const T *qrow = (const T *)p.q + b * p.qs.b + h * p.qs.h + (int64_t)row * p.qs.s;
    const T *orow = (const T *)p.out + b * p.os.b + h * p.os.h + (int64_t)row * p.os.s;
    const T *grow = (const T *)p.dout + b * p.dos.b + h * p.dos.h + (int64_t)row * p.dos.s;
    const T *kbase = (const T *)p.k + b * p.ks.b + hk * p.ks.h;
    const T *vbase = (const T *)p.v + b * p.vs.b + hk * p.vs.h;
    frag qf[C], gf[C];
    float delta = 0.f;
#pragma unroll
    for (int c = 0; c < C; c++) {
        union { ux4 u; frag f; } x, g, o;
        x.u = load_chunk<T>(qrow, 2 * c + half, p.d, live, p.vec);
        g.u = load_chunk<T>(grow, 2 * c + half, p.dv_d, live, p.vec);
        o.u = load_chunk<T>(orow, 2 * c + half, p.dv_d, live, p.vec);
        qf[c] = x.f;
        gf[c] = g.f;
#pragma unroll
        for (int i = 0; i < AT::E; i++) delta += (float)g.f[i] * (float)o.f[i];
    }
    delta += other_half(delta);
    const int64_t stat = ((int64_t)b * p.hq + h) * p.sq + row;
    float lse = kInf;                                              // a row that sees nothing, or is none: every p is zero
    if (live) {
        const float x = p.lse[stat];
        lse = x == -kInf ? kInf : x * kScoreUnit;
        if (half == 0) p.delta[stat] = delta;
    }

    int dq_id = 0, w_lo = 0, w_hi = 0;
    int2 wg_span = {0, 0};
    const int *docs = p.docs != nullptr ? p.docs + b * p.docs_b : nullptr;
    const int2 *ranges = p.doc_range + (int64_t)b * p.doc_blocks;
    if (threadIdx.x == 0) lds_bad = -1;
    if (docs != nullptr) {
        const int raw = live ? max(docs[pos], -1) : -1;
        w_lo = wave_min(raw);
        w_hi = wave_max(raw);
        if (lane == 0) { lds_doc[wave] = w_lo; lds_doc[4 + wave] = w_hi; }
        dq_id = raw < 0 ? -2 : raw;
        __syncthreads();
        wg_span.x = min(min(lds_doc[0], lds_doc[1]), min(lds_doc[2], lds_doc[3]));
        wg_span.y = max(max(lds_doc[4], lds_doc[5]), max(lds_doc[6], lds_doc[7]));
    }
    const int key_end = p.causal ? max(min(pos_end, p.sk), prefix) : p.sk;
    const int tiles = key_end > 0 ? (key_end + TK - 1) / TK : 0;

    fx16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) acc[db] = fx16{};
    float dslope = 0.f;

    for (int base = 0; base < tiles; base += 64) {
        bool want = base + lane < tiles;
        if (docs != nullptr && want) {
            const int k0 = (base + lane) * TK;
            want = docs_meet(doc_span(ranges, k0, min(k0 + TK, p.sk)), wg_span);
        }
        for (uint64_t todo = __ballot(want); todo != 0; todo &= todo - 1) {
            const int tile = base + __builtin_ctzll(todo), k0 = tile * TK, rows = min(TK, p.sk - k0);
            bool doc_full = true, wave_doc_full = true;
            if (docs != nullptr) {
                const int2 s = doc_span(ranges, k0, k0 + rows);
                doc_full = s.x == s.y && s.x >= 0 && wg_span.x == s.x && wg_span.y == s.x;
                wave_doc_full = s.x == s.y && s.x >= 0 && w_lo == s.x && w_hi == s.x;
            }
            const bool in_prefix = k0 + TK <= prefix;
            const bool whole = rows == TK && doc_full && (!p.causal || in_prefix || k0 + TK - 1 <= i0 + off);
            const bool full = rows == TK && wave_doc_full && (!p.causal || in_prefix || k0 + TK - 1 <= pos_lo);
            Stage<T, DP, TK> sk, sv;
            sk.load(kbase + (int64_t)k0 * p.ks.s, p.ks.s, rows, p.d, p.vec);
            sv.load(vbase + (int64_t)k0 * p.vs.s, p.vs.s, rows, p.dv_d, p.vec);
            __syncthreads();
            sk.store(lds_k);
            sv.store(lds_v);
            if (!whole && sk.nonfinite()) lds_bad = tile;
            __syncthreads();
            const bool careful = !whole && lds_bad == tile;
            if (p.causal && k0 > pos_lo + 31 && k0 >= prefix) continue;
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                fx16 s = {}, dp = {};
#pragma unroll
                for (int c = 0; c < C; c++) {
                    s = AT::mma(TL::rows(lds_k, 32 * kb, c), qf[c], s);
                    dp = AT::mma(TL::rows(lds_v, 32 * kb, c), gf[c], dp);
                }
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = k0 + 32 * kb + 8 * (r >> 2) + 4 * half + (r & 3);
                    float t = 0.f;
                    const float x = score<T, MOD>(p, s[r], slope, pos, key, t);
                    float g = __builtin_amdgcn_exp2f(x - lse) * (dp[r] - delta);
                    bool see = live;
                    if (!full) {
                        see = see && key < p.sk && (!p.causal || key <= pos || key < prefix);
                        if (docs != nullptr) see = see && docs[min(key, p.sk - 1)] == dq_id;
                    }
                    g = see ? g : 0.f;
                    if (MOD) {
                        dslope -= g * __builtin_fabsf((float)(pos - key));
                        if (p.cap > 0.f) g *= 1.f - t * t;
                    }
                    s[r] = g;
                }
#pragma unroll
                for (int st = 0; st < ST; st++) {
                    const frag gfr = pack<T>(s, st);
#pragma unroll
                    for (int db = 0; db < DB; db++) {
                        const frag kf = TL::cols(lds_k, 32 * kb + AT::KS * st, 32 * db);
                        if (careful) acc[db] = mma_careful<T>(kf, gfr, acc[db]);
                        else acc[db] = AT::mma(kf, gfr, acc[db]);
                    }
                }
            }
        }
    }
    if (MOD && p.dslopes_part != nullptr) {                        // in a fixed order: lanes, then waves
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) dslope += __shfl_xor(dslope, o, 64);
        if (lane == 0) lds_sum[wave] = dslope;
        __syncthreads();
        if (threadIdx.x == 0)
            p.dslopes_part[((int64_t)h * p.b + b) * tiles_q + tile_q] = (lds_sum[0] + lds_sum[1]) + (lds_sum[2] + lds_sum[3]);
    }
    if (!live || p.dq == nullptr) return;
    T *out = (T *)p.dq + (((int64_t)b * p.sq + row) * p.hq + h) * p.d;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int c = 32 * db + 8 * (r >> 2) + 4 * half + (r & 3);
            if (c < p.d) out[c] = (T)(acc[db][r] * p.scale);
        }
}

template <typename T, int DP, bool MOD>
__global__ void __launch_bounds__(kAttnThreads, 1) attention_dkv_kernel(AttnArgs p) {
    typedef AttnType<T> AT;
    typedef typename AT::frag frag;
    typedef Tile<T, DP> TL;
    constexpr int TQ = AT::kTile, QB = TQ / 32, C = DP / AT::KS, DB = DP / 32, ST = 32 / AT::KS;
    __shared__ __align__(16) char lds_q[TQ * TL::RB];
    __shared__ __align__(16) char lds_g[TQ * TL::RB];
    __shared__ float lds_lse[TQ], lds_delta[TQ];
    __shared__ int lds_id[TQ];
    __shared__ int lds_doc[8];
    __shared__ int lds_bad;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int pairs = p.b * p.hk, tiles_k = (p.sk + kAttnRows - 1) / kAttnRows;
    const int pair = blockIdx.x % pairs, split = blockIdx.x / pairs % p.splits, tile_k = blockIdx.x / pairs / p.splits;
    const int b = pair / p.hk, hk = pair % p.hk;
    const int off = p.sk - p.sq;
    const int k0 = tile_k * kAttnRows, key = k0 + wave * 32 + (lane & 31);
    const bool live = key < p.sk;
    const int k_lo = k0 + wave * 32;
    const int prefix = p.prefix != nullptr ? min(p.prefix[b], p.sk) : 0;

    const T *krow = (const T *)p.k + b * p.ks.b + hk * p.ks.h + (int64_t)key * p.ks.s;
    const T *vrow = (const T *)p.v + b * p.vs.b + hk * p.vs.h + (int64_t)key * p.vs.s;
    frag kf[C], vf[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        union { ux4 u; frag f; } x, y;
        x.u = load_chunk<T>(krow, 2 * c + half, p.d, live, p.vec);
        y.u = load_chunk<T>(vrow, 2 * c + half, p.dv_d, live, p.vec);
        kf[c] = x.f;
        vf[c] = y.f;
    }
    int key_id = 0, w_lo = 0, w_hi = 0;
    int2 wg_span = {0, 0};
    const int *docs = p.docs != nullptr ? p.docs + b * p.docs_b : nullptr;
    const int2 *ranges = p.doc_range + (int64_t)b * p.doc_blocks;
    if (threadIdx.x == 0) lds_bad = -1;
    if (docs != nullptr) {
        const int raw = live ? max(docs[key], -1) : -1;
        w_lo = wave_min(raw);
        w_hi = wave_max(raw);
        if (lane == 0) { lds_doc[wave] = w_lo; lds_doc[4 + wave] = w_hi; }
        key_id = raw < 0 ? -2 : raw;
        __syncthreads();
        wg_span.x = min(min(lds_doc[0], lds_doc[1]), min(lds_doc[2], lds_doc[3]));
        wg_span.y = max(max(lds_doc[4], lds_doc[5]), max(lds_doc[6], lds_doc[7]));
    }
    // rows that may see a key of this tile: with the causal mask those at or behind its first key, or all for a prefix
    const int first = p.causal && k0 >= prefix ? max(k0 - off, 0) : 0;
    const int tile_lo = first / TQ, tile_hi = (p.sq + TQ - 1) / TQ;

    fx16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) dk[db] = dv[db] = fx16{};

    const int h_lo = p.group * split / p.splits, h_hi = p.group * (split + 1) / p.splits;
    for (int hg = h_lo; hg < h_hi; hg++) {
        const int h = hk * p.group + hg;
        const float slope = MOD && p.slopes != nullptr ? p.slopes[h] : 0.f;
        const T *qbase = (const T *)p.q + b * p.qs.b + h * p.qs.h;
        const T *gbase = (const T *)p.dout + b * p.dos.b + h * p.dos.h;
        const int64_t stat = ((int64_t)b * p.hq + h) * p.sq;
        for (int base = tile_lo; base < tile_hi; base += 64) {
            bool want = base + lane < tile_hi;
            if (docs != nullptr && want) {
                const int lo = (base + lane) * TQ;
                want = docs_meet(doc_span(ranges, lo + off, min(lo + TQ, p.sq) + off), wg_span);
            }
            for (uint64_t todo = __ballot(want); todo != 0; todo &= todo - 1) {
                const int tile = base + __builtin_ctzll(todo), i0 = tile * TQ, rows = min(TQ, p.sq - i0);
                bool doc_full = true, wave_doc_full = true;
                if (docs != nullptr) {
                    const int2 s = doc_span(ranges, i0 + off, i0 + rows + off);
                    doc_full = s.x == s.y && s.x >= 0 && wg_span.x == s.x && wg_span.y == s.x;
                    wave_doc_full = s.x == s.y && s.x >= 0 && w_lo == s.x && w_hi == s.x;
                }
                const bool whole = rows == TQ && doc_full && (!p.causal || k0 + kAttnRows - 1 <= i0 + off || k0 + kAttnRows <= prefix);
                const bool full = rows == TQ && wave_doc_full && (!p.causal || k_lo + 31 <= i0 + off || k_lo + 32 <= prefix);
                Stage<T, DP, TQ> sq, sg;
                sq.load(qbase + (int64_t)i0 * p.qs.s, p.qs.s, rows, p.d, p.vec);
                sg.load(gbase + (int64_t)i0 * p.dos.s, p.dos.s, rows, p.dv_d, p.vec);
                float r_lse = kInf, r_delta = 0.f;
                int r_id = -1;
                if ((int)threadIdx.x < rows) {
                    const float x = p.lse[stat + i0 + threadIdx.x];
                    r_lse = x == -kInf ? kInf : x * kScoreUnit;
                    r_delta = p.delta[stat + i0 + threadIdx.x];
                    if (docs != nullptr) r_id = max(docs[i0 + threadIdx.x + off], -1);
                }
                __syncthreads();
                sq.store(lds_q);
                sg.store(lds_g);
                if (threadIdx.x < TQ) { lds_lse[threadIdx.x] = r_lse; lds_delta[threadIdx.x] = r_delta; lds_id[threadIdx.x] = r_id; }
                const int seq = hg * tile_hi + tile;
                if (!whole && (sq.nonfinite() || sg.nonfinite())) lds_bad = seq;
                __syncthreads();
                const bool careful = !whole && lds_bad == seq;
                if (p.causal && k_lo > i0 + TQ - 1 + off && k_lo >= prefix) continue;
#pragma unroll
                for (int qb = 0; qb < QB; qb++) {
                    fx16 s = {}, dp = {};
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        s = AT::mma(TL::rows(lds_q, 32 * qb, c), kf[c], s);
                        dp = AT::mma(TL::rows(lds_g, 32 * qb, c), vf[c], dp);
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int at = 32 * qb + 8 * (r >> 2) + 4 * half + (r & 3), i = i0 + at, pos = i + off;
                        float t = 0.f;
                        const float x = score<T, MOD>(p, s[r], slope, pos, key, t);
                        float e = __builtin_amdgcn_exp2f(x - lds_lse[at]);
                        float g = e * (dp[r] - lds_delta[at]);
                        bool see = live;
                        if (!full) {
                            see = see && i < p.sq && (!p.causal || key <= pos || key < prefix);
                            if (docs != nullptr) see = see && lds_id[at] == key_id;
                        }
                        if (MOD && p.cap > 0.f) g *= 1.f - t * t;
                        s[r] = see ? e : 0.f;
                        dp[r] = see ? g : 0.f;
                    }
#pragma unroll
                    for (int st = 0; st < ST; st++) {
                        const frag pf = pack<T>(s, st), sf = pack<T>(dp, st);
#pragma unroll
                        for (int db = 0; db < DB; db++) {
                            const frag gt = TL::cols(lds_g, 32 * qb + AT::KS * st, 32 * db);
                            const frag qt = TL::cols(lds_q, 32 * qb + AT::KS * st, 32 * db);
                            if (careful) {
                                dv[db] = mma_careful<T>(gt, pf, dv[db]);
                                dk[db] = mma_careful<T>(qt, sf, dk[db]);
                            } else {
                                dv[db] = AT::mma(gt, pf, dv[db]);
                                dk[db] = AT::mma(qt, sf, dk[db]);
                            }
                        }
                    }
                }
            }
        }
    }
    if (!live) return;
    const int64_t at_k = (((int64_t)b * p.sk + key) * p.hk + hk) * p.d, at_v = (((int64_t)b * p.sk + key) * p.hk + hk) * p.dv_d;
    if (p.splits == 1) {
        T *ok = (T *)p.dk + at_k, *ov = (T *)p.dv + at_v;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = 32 * db + 8 * (r >> 2) + 4 * half + (r & 3);
                if (c < p.d) ok[c] = (T)(dk[db][r] * p.scale);
                if (c < p.dv_d) ov[c] = (T)dv[db][r];
            }
    } else {                                                       // parts in float, added by attention_join_kernel
        const int64_t nk = (int64_t)p.b * p.sk * p.hk * p.d, nv = (int64_t)p.b * p.sk * p.hk * p.dv_d;
        float *ok = p.dkv_part + split * nk + at_k, *ov = p.dkv_part + p.splits * nk + split * nv + at_v;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = 32 * db + 8 * (r >> 2) + 4 * half + (r & 3);
                if (c < p.d) ok[c] = dk[db][r] * p.scale;
                if (c < p.dv_d) ov[c] = dv[db][r];
            }
    }
}

template <typename T> int launch_attention_dq(const AttnArgs &a, int dp, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.b * a.hq * ((a.sq + kAttnRows - 1) / kAttnRows)));
    FLK_ATTN_LAUNCH(attention_dq_kernel, grid)
}
template <typename T> int launch_attention_dkv(const AttnArgs &a, int dp, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.b * a.hk * a.splits * ((a.sk + kAttnRows - 1) / kAttnRows)));
    FLK_ATTN_LAUNCH(attention_dkv_kernel, grid)
}
template int launch_attention_dq<attn_t>(const AttnArgs &, int, hipStream_t);
template int launch_attention_dkv<attn_t>(const AttnArgs &, int, hipStream_t);

}  // namespace flk
