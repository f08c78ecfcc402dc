// Attention of the newest tokens of ragged sequences over a cache of keys and values (gfx950).  Compiled once per element type.
//
// Bound by reading the cache once.  The query rows that read the same keys (the heads that share a key head, times the new
// tokens) are packed into the 32 columns of the matrix instructions, so that products cost little beside the reads, and the
// keys of a sequence are divided over workgroups and over a workgroup's four or eight waves.  Every wave walks over tiles of 32 keys of
// its own with no barrier: the next tile's reads are in flight, in registers, while the present one is used from LDS.  The waves'
// results meet in LDS, those of several workgroups in a second kernel, both in a fixed order.
#include "attention_common.h"

namespace flk {

template <typename T, int DP, int MOD, int W>
__global__ void __launch_bounds__(64 * W, W > 4 || (sizeof(T) == 4 && DP > 64) ? 1 : 2) attention_cached_kernel(CachedArgs p) {
    typedef AttnType<T> AT;
    typedef typename AT::frag frag;
    typedef Tile<T, DP> TL;
    constexpr int TK = kCachedKeys, C = DP / AT::KS, DB = DP / 32, ST = 32 / AT::KS, NC = TL::NC, N = TK * NC / 64;
    constexpr int kWave = 2 * TK * TL::RB, kJoin = 32 * (DP + 1) * 4;          // LDS of a wave: its tiles, later its output
    constexpr int kLds = kWave > kJoin ? kWave : kJoin;
    __shared__ __align__(16) char lds[W * kLds];
    __shared__ float lds_ml[W][32][2];
    static_assert(W * (kLds + 256) <= 160 * 1024, "LDS of a workgroup");

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int pairs = p.b * p.hk;
    const int pair = blockIdx.x % pairs, rest = blockIdx.x / pairs, rb = rest % p.blocks_r, split = rest / p.blocks_r;
    const int b = pair / p.hk, hk = pair % p.hk;
    const int len = max(0, min(p.lengths[b], p.capacity));
    const int n_rows = p.t * p.group;
    const int r = rb * 32 + (lane & 31);
    const bool live = r < n_rows;
    const int t = r / p.group, h = hk * p.group + r % p.group;
    const int pos = len - p.t + t, pos_lo = len - p.t + rb * 32 / p.group;
    const Score<T, MOD> score(p.scale, p.cap, (MOD & kDecay) && p.slopes != nullptr && live ? p.slopes[h] : 0.f);
    // this workgroup's keys, in whole tiles
    const int all = (len + TK - 1) / TK, per = (all + p.splits - 1) / p.splits;
    const int tile_lo = min(split * per, all), tile_hi = min(tile_lo + per, all);

    const T *qrow = (const T *)p.q + b * p.qs.b + (int64_t)t * p.qs.s + h * p.qs.h;
    const T *kbase = (const T *)p.k + b * p.ks.b + hk * p.ks.h;
    const T *vbase = (const T *)p.v + b * p.vs.b + hk * p.vs.h;
    char *lds_k = lds + wave * kLds, *lds_v = lds_k + TK * TL::RB;
    typename TL::Lane at_lane;
    at_lane.init();
    frag qf[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        union { ux4 u; frag f; } x;
        x.u = load_chunk<T>(qrow, 2 * c + half, p.d, live, p.vec);
        qf[c] = x.f;
    }
    fx16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) o[db] = fx16{};
    float m = -kInf, l = 0.f;

    ux4 rk[N], rv[N];
    auto fetch = [&](int tile) {
        const int k0 = tile * TK;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int i = n * 64 + lane, row = k0 + i / NC, c = i % NC;
            rk[n] = load_chunk<T>(kbase + row * p.ks.s, c, p.d, row < len, p.vec);
            rv[n] = load_chunk<T>(vbase + row * p.vs.s, c, p.dv_d, row < len, p.vec);
        }
    };
    int tile = tile_lo + wave;
    if (tile < tile_hi) fetch(tile);
    for (; tile < tile_hi; tile += W) {
        const int k0 = tile * TK;
        const bool full = k0 + TK - 1 <= pos_lo;
        bool bad = false;
        if (!full) {
#pragma unroll
            for (int n = 0; n < N; n++) bad |= any_nonfinite<T>(rv[n]);
        }
        const bool careful = !full && __any(bad);
        if (careful) {                                             // clear them for the product, and add what they do to it below
#pragma unroll
            for (int n = 0; n < N; n++) rv[n] = cleaned<T>(rv[n]); // (here, not in LDS: there a lane's 16 bytes are another lane's)
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int i = n * 64 + lane, row = i / NC, c = i % NC;
            *(ux4 *)(lds_k + TL::at(row, c)) = rk[n];
            *(ux4 *)(lds_v + TL::at(row, c)) = rv[n];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (tile + W < tile_hi) fetch(tile + W);
        fx16 s = {};
#pragma unroll
        for (int c = 0; c < C; c++) s = AT::mma(TL::rows(lds_k, at_lane, 0, c), qf[c], s);
        float top = -kInf;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int key = k0 + 8 * (i >> 2) + 4 * half + (i & 3);
            float grad, x = score(s[i], (float)(pos - key), grad);
            if (!full) x = key <= pos ? x : -kInf;                 // pos < len: nothing behind the sequence either
            s[i] = x;
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
        constexpr float kLift = kNarrow<T> ? 14.f : 0.f;           // (the same for all parts: their maxima join them as they are)
        const float base_m = m == -kInf ? 0.f : m - kLift;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = __builtin_amdgcn_exp2f(s[i] - base_m);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};                       // short chains: long ones would cost float data digits
#pragma unroll
        for (int i = 0; i < 16; i++) sum[i & 3] += s[i];
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int st = 0; st < ST; st++) {
            // 16-bit weights are rounded once, as in the other kernels.  (In two pieces, the second holding what rounding took from the first,
            // results are those of 32 bits, 1.67e-3 from the exact ones where these are 1.81e-3, almost all of it their own rounding;
            // 64 sequences of up to 16 384 keys take 510 us so instead of 434.)
            const frag pf = pack<T>(s, st);
#pragma unroll
            for (int db = 0; db < DB; db++) {
                const frag vf = TL::cols(lds_v, at_lane, AT::KS * st, db);
                o[db] = AT::mma(vf, pf, o[db]);
            }
        }
        if (careful) {
            fx16 x[DB];
#pragma unroll
            for (int db = 0; db < DB; db++) x[db] = o[db];
            spread_nonfinite<T, TK, DB>(vbase + k0 * p.vs.s, p.vs.s, len - k0, p.dv_d, seen_from(low_bits(pos + 1 - k0)), 1.f, x);
#pragma unroll
            for (int db = 0; db < DB; db++) o[db] = x[db];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    l += other_half(l);

    // the waves' results: o relative to the largest of their maxima
    float *mine = (float *)(lds + wave * kLds);
    __syncthreads();
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int i = 0; i < 16; i++) mine[(lane & 31) * (DP + 1) + 32 * db + 8 * (i >> 2) + 4 * half + (i & 3)] = o[db][i];
    if (half == 0) { lds_ml[wave][lane][0] = m; lds_ml[wave][lane][1] = l; }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * DP; i += 64 * W) {
        const int rr = i / DP, c = i % DP, row = rb * 32 + rr;
        if (row >= n_rows || c >= p.dv_d) continue;
        float top = lds_ml[0][rr][0];
#pragma unroll
        for (int w = 1; w < W; w++) top = fmaxf(top, lds_ml[w][rr][0]);
        float x = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float mw = lds_ml[w][rr][0];
            if (mw == -kInf && lds_ml[w][rr][1] == 0.f) continue;  // saw nothing
            const float a = mw == -kInf ? 1.f : __builtin_amdgcn_exp2f(mw - top);
            x += a * ((const float *)(lds + w * kLds))[rr * (DP + 1) + c];
            sum += a * lds_ml[w][rr][1];
        }
        const int tt = row / p.group, hh = hk * p.group + row % p.group;
        const int64_t at = ((int64_t)b * p.t + tt) * p.hq + hh;
        if (p.splits == 1) ((T *)p.out)[at * p.dv_d + c] = (T)(sum == 0.f ? 0.f : x / sum);
        else {
            p.part_o[(at * p.splits + split) * p.dv_d + c] = x;
            if (c == 0) { p.part_ml[(at * p.splits + split) * 2] = top; p.part_ml[(at * p.splits + split) * 2 + 1] = sum; }
        }
    }
}

// out from the parts of `splits` workgroups: a workgroup a row.  The parts' shares first, one thread each; then threads in groups
// that hold the row's values add the parts, every group each `groups`-th one, and the groups' sums meet in LDS.
constexpr int kMaxSplits = 256;
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) attention_cached_join_kernel(CachedArgs p) {
    __shared__ float share[kMaxSplits], sums[THREADS], lds_top[THREADS / 64], lds_sum[THREADS / 64];
    const int64_t row = blockIdx.x;
    const float *ml = p.part_ml + row * p.splits * 2, *po = p.part_o + row * p.splits * p.dv_d;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float top = -kInf;
    for (int s = threadIdx.x; s < p.splits; s += THREADS) top = fmaxf(top, ml[2 * s]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (lane == 0) lds_top[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) top = fmaxf(top, lds_top[w]);
    float sum = 0.f;
    for (int s = threadIdx.x; s < p.splits; s += THREADS) {
        const float m = ml[2 * s], l = ml[2 * s + 1];
        // a part that saw nothing has no share; one whose scores were all NaN has a maximum of -inf and a sum of NaN
        const float a = m == -kInf ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - top);
        share[s] = a;
        sum += a * l;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) lds_sum[wave] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) sum += lds_sum[w];
    int width = 32;
    while (width < p.dv_d) width *= 2;                             // at most 128, the padded head
    const int c = threadIdx.x % width, group = threadIdx.x / width, groups = THREADS / width;
    float x = 0.f;
    if (c < p.dv_d) {
#pragma unroll 8
        for (int s = group; s < p.splits; s += groups)
            if (share[s] != 0.f) x += share[s] * po[(int64_t)s * p.dv_d + c];
    }
    sums[threadIdx.x] = x;
    __syncthreads();
    if (group != 0 || c >= p.dv_d) return;
    x = 0.f;
    for (int g = 0; g < groups; g++) x += sums[g * width + c];
    ((T *)p.out)[row * p.dv_d + c] = (T)(sum == 0.f ? 0.f : x / sum);
}

template <typename T, int DP, int W> void launch_cached_waves(const CachedArgs &a, int kind, dim3 grid, hipStream_t st) {
    if (kind == kPlain) hipLaunchKernelGGL((attention_cached_kernel<T, DP, kPlain, W>), grid, dim3(64 * W), 0, st, a);
    else if (kind == kCap) hipLaunchKernelGGL((attention_cached_kernel<T, DP, kCap, W>), grid, dim3(64 * W), 0, st, a);
    else if (kind == kDecay) hipLaunchKernelGGL((attention_cached_kernel<T, DP, kDecay, W>), grid, dim3(64 * W), 0, st, a);
    else hipLaunchKernelGGL((attention_cached_kernel<T, DP, kCapDecay, W>), grid, dim3(64 * W), 0, st, a);
}
template <typename T, int DP> void launch_cached_kind(const CachedArgs &a, int kind, dim3 grid, hipStream_t st) {
    constexpr bool kRoom = sizeof(T) == 2 || DP <= 64;             // eight waves' tiles fit into 160 KB of LDS
    if constexpr (kRoom) {
        if (a.waves == 8) { launch_cached_waves<T, DP, 8>(a, kind, grid, st); return; }
    }
    launch_cached_waves<T, DP, 4>(a, kind, grid, st);
}

template <typename T> int launch_attention_cached(const CachedArgs &a, int dp, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.b * a.hk * a.blocks_r * a.splits));
    const int kind = score_kind(a.scale, a.cap, a.slopes);
    if (dp == 32) launch_cached_kind<T, 32>(a, kind, grid, st);
    else if (dp == 64) launch_cached_kind<T, 64>(a, kind, grid, st);
    else if (dp == 96) launch_cached_kind<T, 96>(a, kind, grid, st);
    else launch_cached_kind<T, 128>(a, kind, grid, st);
    FLK_LAUNCH_CHECK("attention_cached_kernel");
    if (a.splits > 1) {
        const dim3 rows((unsigned)((int64_t)a.b * a.t * a.hq));
        if (a.splits > 16) hipLaunchKernelGGL((attention_cached_join_kernel<T, 1024>), rows, dim3(1024), 0, st, a);
        else hipLaunchKernelGGL((attention_cached_join_kernel<T, 128>), rows, dim3(128), 0, st, a);
        FLK_LAUNCH_CHECK("attention_cached_join_kernel");
    }
    return FLK_OK;
}
template int launch_attention_cached<attn_t>(const CachedArgs &, int, hipStream_t);

}  // namespace flk
