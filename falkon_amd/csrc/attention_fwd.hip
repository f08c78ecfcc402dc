// Attention, forward: one pass over the keys with a running maximum and sum (gfx950).  Compiled once per element type.
//
// A workgroup owns 128 queries of one head, a wave 32 of them, with its queries and its 32 x d output in registers; tiles of
// keys and values go through LDS.  The maximum is kept per row and the output rescaled only when some row of the wave found a
// larger one.  Keys, values and probabilities never leave the chip.
#include "attention_common.h"

namespace flk {

template <typename T, int DP, bool MOD>
__global__ void __launch_bounds__(kAttnThreads, 2) attention_fwd_kernel(AttnArgs p) {
    typedef AttnType<T> AT;
    typedef typename AT::frag frag;
    typedef Tile<T, DP> TL;
    constexpr int TK = AT::kTile, KB = TK / 32, C = DP / AT::KS, DB = DP / 32, ST = 32 / AT::KS;
    __shared__ __align__(16) char lds_k[TK * TL::RB];
    __shared__ __align__(16) char lds_v[TK * TL::RB];
    __shared__ int lds_doc[8];
    __shared__ int lds_bad;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    // consecutive workgroups go to different XCDs: heads that share keys stay on one of them, the longest rows go first
    const int heads = p.b * p.hq, pairs = p.b * p.hk;
    const int hb = blockIdx.x % heads, tiles_q = (p.sq + kAttnRows - 1) / kAttnRows;
    const int tile_q = tiles_q - 1 - blockIdx.x / heads;
    const int b = hb % pairs / p.hk, hk = hb % p.hk, h = hk * p.group + hb / pairs;
    const int off = p.sk - p.sq;
    const int i0 = tile_q * kAttnRows, row = i0 + wave * 32 + (lane & 31);
    const bool live = row < p.sq;
    const int pos = row + off;
    const int pos_lo = i0 + wave * 32 + off;                       // first position of this wave
    const int pos_end = min(i0 + kAttnRows, p.sq) + off;           // behind the last position of the workgroup
    const float slope = MOD && p.slopes != nullptr ? p.slopes[h] : 0.f;
    const int prefix = p.prefix != nullptr ? min(p.prefix[b], p.sk) : 0;

    const T *qrow = (const T *)p.q + b * p.qs.b + h * p.qs.h + (int64_t)row * p.qs.s;
    const T *kbase = (const T *)p.k + b * p.ks.b + hk * p.ks.h;
    const T *vbase = (const T *)p.v + b * p.vs.b + hk * p.vs.h;
    frag qf[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        union { ux4 u; frag f; } x;
        x.u = load_chunk<T>(qrow, 2 * c + half, p.d, live, p.vec);
        qf[c] = x.f;
    }

    // documents: this row's id (no key has -2) and the span of the wave's and of the workgroup's rows
    int dq = 0, w_lo = 0, w_hi = 0;
    int2 wg_span = {0, 0};
    const int *docs = p.docs != nullptr ? p.docs + b * p.docs_b : nullptr;
    const int2 *ranges = p.doc_range + (int64_t)b * p.doc_blocks;
    if (threadIdx.x == 0) lds_bad = -1;
    if (docs != nullptr) {
        const int raw = live ? max(docs[pos], -1) : -1;
        w_lo = wave_min(raw);
        w_hi = wave_max(raw);
        if (lane == 0) { lds_doc[wave] = w_lo; lds_doc[4 + wave] = w_hi; }
        dq = raw < 0 ? -2 : raw;
        __syncthreads();
        wg_span.x = min(min(lds_doc[0], lds_doc[1]), min(lds_doc[2], lds_doc[3]));
        wg_span.y = max(max(lds_doc[4], lds_doc[5]), max(lds_doc[6], lds_doc[7]));
    }

    const int key_end = p.causal ? max(min(pos_end, p.sk), prefix) : p.sk;
    const int tiles = key_end > 0 ? (key_end + TK - 1) / TK : 0;

    fx16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) o[db] = fx16{};
    float m = -kInf, l = 0.f;

    for (int base = 0; base < tiles; base += 64) {
        bool want = base + lane < tiles;
        if (docs != nullptr && want) {
            const int k0 = (base + lane) * TK;
            want = docs_meet(doc_span(ranges, k0, min(k0 + TK, p.sk)), wg_span);
        }
        for (uint64_t todo = __ballot(want); todo != 0; todo &= todo - 1) {
            const int tile = base + __builtin_ctzll(todo), k0 = tile * TK, rows = min(TK, p.sk - k0);
            // whether this tile needs no mask, for the workgroup (causal side: its first row) and for this wave
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
            __syncthreads();                                       // the previous tile has been read
            sk.store(lds_k);
            sv.store(lds_v);
            if (!whole && sv.nonfinite()) lds_bad = tile;
            __syncthreads();
            const bool careful = !whole && lds_bad == tile;
            // a wave none of whose rows sees anything here
            if (p.causal && k0 > pos_lo + 31 && k0 >= prefix) continue;

            fx16 s[KB];
            float top = -kInf;
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                s[kb] = fx16{};
#pragma unroll
                for (int c = 0; c < C; c++) s[kb] = AT::mma(TL::rows(lds_k, 32 * kb, c), qf[c], s[kb]);
            }
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = k0 + 32 * kb + 8 * (r >> 2) + 4 * half + (r & 3);
                    float t, x = score<T, MOD>(p, s[kb][r], slope, pos, key, t);
                    if (!full) {
                        bool see = key < p.sk && (!p.causal || key <= pos || key < prefix);
                        if (docs != nullptr) see = see && docs[min(key, p.sk - 1)] == dq;
                        x = see ? x : -kInf;
                    }
                    s[kb][r] = x;
                    top = fmaxf(top, x);
                }
            top = fmaxf(top, other_half(top));
            if (__any(top > m)) {
                const float next = fmaxf(m, top);
                const float a = m == -kInf ? 0.f : __builtin_amdgcn_exp2f(m - next);
                l *= a;
                m = next;
#pragma unroll
                for (int db = 0; db < DB; db++) o[db] *= a;
            }
            const float base_m = m == -kInf ? 0.f : m;
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[kb][r] = __builtin_amdgcn_exp2f(s[kb][r] - base_m);
                    l += s[kb][r];
                }
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int st = 0; st < ST; st++) {
                    const frag pf = pack<T>(s[kb], st);
#pragma unroll
                    for (int db = 0; db < DB; db++) {
                        const frag vf = TL::cols(lds_v, 32 * kb + AT::KS * st, 32 * db);
                        if (careful) o[db] = mma_careful<T>(vf, pf, o[db]);
                        else o[db] = AT::mma(vf, pf, o[db]);
                    }
                }
        }
    }
    l += other_half(l);
    if (!live) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;                    // a row that sees nothing is zero
    T *orow = (T *)p.o + (((int64_t)b * p.sq + row) * p.hq + h) * p.dv_d;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int c = 32 * db + 8 * (r >> 2) + 4 * half + (r & 3);
            if (c < p.dv_d) orow[c] = (T)(o[db][r] * inv);
        }
    if (half == 0 && p.lse != nullptr)
        p.lse[((int64_t)b * p.hq + h) * p.sq + row] = l == 0.f ? -kInf : m * kLn2 + __logf(l);
}

template <typename T> int launch_attention_fwd(const AttnArgs &a, int dp, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.b * a.hq * ((a.sq + kAttnRows - 1) / kAttnRows)));
    FLK_ATTN_LAUNCH(attention_fwd_kernel, grid)
}
template int launch_attention_fwd<attn_t>(const AttnArgs &, int, hipStream_t);

}  // namespace flk
