// Verification of drafted tokens (speculative decoding by rejection): ifh_verify_drafts_f32 on whole distributions,
// ifh_verify_drafts_topk on the top-k sampler's candidates.
//
// The draw compares a cumulated mass with a given number, and a vocabulary of 150 000 tokens has borders 1e-6 apart: masses are f64 to
// their last bits, so that neither the way a sum is split nor the exponential's rounding moves a border past the number (f32 exponentials
// would move one in every few hundred draws from a flat tail).  The f64 work (17 operations a logit) stays just under the time the logits
// take to arrive.
//   k_verify_stats   a wave or four a chunk of a target row: (max, sum of exp), or the arg-max for temperature 0.  Bound by memory: 320 rows of
//                    151 936 logits, 194 MB, 41 us = 4.7 TB/s
//   k_verify_mass    a wave or four a chunk of the refused position, where the draft has a distribution: the mass of max(p - q, 0).  64 rows of both,
//                    78 MB, 15.5 us, 4 of them for the verdicts in front
//   k_verify_draw    a workgroup a row: the chunk and then the token where the cumulated mass passes the uniform number.  A chain of
//                    dependent loads and scans, 6.4 us for one row and 6.0 for 64
// A chunk is 2048 logits: one row of 151 936 is 75 of them, so that one call's few rows still spread over the device.
#include "common.h"

namespace ifh {

constexpr int VT = 256, VPL = 32, VC = 64 * VPL;        // threads, logits a lane, logits a chunk (a wave's)
constexpr int VM = 512, VD = 512;                       // threads of the mass and the draw launch (draw: 1024 0.35 us more, 256 0.5 us)
constexpr int kVerifyMaxChunks = 256;                   // 524 288 tokens: the draw gives each chunk a thread
constexpr float kFltMax = 3.402823466e38f;

// 2^(j / 32)
__device__ const double kExp2[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
    1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951, 1.4451808069770467,
    1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649,
    1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103,
    1.9152065613971474, 1.9571441241754002
};
// 32 / (ln 2 temperature), and the difference of logits below which an exponential is 0
struct Rate {
    double rate, least;
};
__device__ __forceinline__ void exp_table(double entry, double (&tab)[32])       // entry: kExp2[threadIdx.x % 32], on its way
{
    if (threadIdx.x < 32) tab[threadIdx.x] = entry;
    __syncthreads();
}
// e^x for x = d / temperature <= 0 in f64; relative error below 4e-16, and what the rate's rounding makes (2.2e-16 |x|).  d rate =
// x 32 / ln 2 = k + u, |u| <= 1/2 (k by adding and taking off 1.5 2^52, the product never rounded), and 2^(k/32) comes from the table (LDS:
// its 32 entries lie in 64 different banks) and k / 32.  e^(u ln 2 / 32) is the Taylor polynomial of degree 6 with u^6 replaced by the
// Chebyshev polynomial's lower terms: degree 5, within 1.5e-16.
__device__ __forceinline__ double exp_neg(double d, const Rate &r, const double (&tab)[32])
{
    const double big = 6755399441055744.0;
    d = fmax(d, r.least);
    const double kb = __builtin_fma(d, r.rate, big), u = __builtin_fma(d, r.rate, big - kb);
    const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, kb);
    double g = __builtin_fma(u, 3.973709984549416e-11, 9.172616498033084e-09);
    g = __builtin_fma(u, g, 1.693850972437182e-06);
    g = __builtin_fma(u, g, 0.0002345961981972034);
    g = __builtin_fma(u, g, 0.02166084939249829);
    const double t = tab[k & 31];
    return __builtin_ldexp(__builtin_fma(t, u * g, t), k >> 5);
}

// NaN counts as -inf; +inf as the largest finite value (its differences stay finite)
__device__ __forceinline__ float logit(float l) { return l == l ? fminf(l, kFltMax) : -INFINITY; }

// which drafts a row keeps, and the statistics of the position that is drawn from
struct Verdict {
    int kept, refused, best;
    float m;
    double s;
};
struct VerifyParams {
    const float *logits;
    int64_t ld;
    const float *q;
    int64_t q_ld;
    const int32_t *drafts, *lens;
    const float *uniform;
    int32_t *out_tokens, *out_count;
    int vocab, T, nch;
    Rate rate;
    int greedy, vec, qvec;
    double *csum;                // [rows * (T+1)][nch] chunk sums of exp((l - cmax) / temperature); greedy: the place of the chunk's maximum
    double *mass;                // [rows][nch]
    float *cmax;                 // [rows * (T+1)][nch] chunk maxima
    Verdict *verdicts;           // [rows], written by the mass launch, or NULL: there is none
};

// a lane's elements of the chunk at `base`: 16 bytes at a time where the row is aligned, else every 64th
__device__ __forceinline__ int place(int vec, int base, int lane, int e) { return base + (vec ? (e >> 2) * 256 + lane * 4 + (e & 3) : e * 64 + lane); }
template <int N>
__device__ __forceinline__ void load_chunk(const float *row, int base, int lane, int vocab, int vec, float fill, float (&v)[N])
{
    if (vec && base + 64 * N <= vocab) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(row + base + e * 64 + lane * 4);
            v[e] = f.x; v[e + 1] = f.y; v[e + 2] = f.z; v[e + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) {
            const int j = place(vec, base, lane, e);
            v[e] = j < vocab ? row[j] : fill;
        }
    }
}

// Scans over the lanes of a wave as DPP operands (shifts by 1, 2, 4, 8 within 16 lanes, then lane 15 of rows 0 and 2 and lane 31 handed
// on): a ds_bpermute step of 64 bits costs two LDS round trips, and the draw is a chain of such scans.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_d(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, true);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double wave_scan_d(double v)
{
    v += dpp_d<0x111, 0xF>(v);
    v += dpp_d<0x112, 0xF>(v);
    v += dpp_d<0x114, 0xF>(v);
    v += dpp_d<0x118, 0xF>(v);
    v += dpp_d<0x142, 0xA>(v);
    v += dpp_d<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ double lane63_d(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double wave_sum_d(double v) { return lane63_d(wave_scan_d(v)); }
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_max(float v)
{
    const int ninf = (int)0xff800000;
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(ninf, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false)));
}
__device__ __forceinline__ float wave_max_f(float v)
{
    v = dpp_max<0x111, 0xF>(v);
    v = dpp_max<0x112, 0xF>(v);
    v = dpp_max<0x114, 0xF>(v);
    v = dpp_max<0x118, 0xF>(v);
    v = dpp_max<0x142, 0xA>(v);
    v = dpp_max<0x143, 0xC>(v);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// W waves a chunk: one (no barrier), or a workgroup's four where there are few chunks for the device, so that a lane has 8 of the f64
// exponentials and not 32.  Four up to 32 chunks a CU: the whole verification of one row of 3 looked-up drafts, 151 936 tokens, 9.7 us (one
// wave a chunk 10.9), of 16 rows of 4 drafts 24.3 us (26.0), of 32 rows 41.5 (41.2), but of 64 rows 69.4 us (64.7).
template <int W> __global__ __launch_bounds__(VT) void k_verify_stats(const VerifyParams p)
{
    constexpr int N = VPL / W;
    __shared__ float ms[W];
    __shared__ double ss[W], tab[32];
    const int64_t pos = blockIdx.y;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int c = W == 1 ? blockIdx.x * 4 + wid : blockIdx.x, base = c * VC + (W == 1 ? 0 : wid * (VC / W));
    const double entry = kExp2[threadIdx.x & 31];
    float v[N];
    load_chunk<N>(p.logits + pos * p.ld, base, lane, p.vocab, p.vec, -INFINITY, v);
    exp_table(entry, tab);
    if (c >= p.nch) return;
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; e++) {
        v[e] = logit(v[e]);
        m = fmaxf(m, v[e]);
    }
    m = wave_max_f(m);
    if (W > 1) {
        if (lane == 0) ms[wid] = m;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < W; k++) m = fmaxf(m, ms[k]);
    }
    double s = 0.0;
    if (p.greedy) {
        int at = 0x7fffffff;                                 // the first place of the maximum
#pragma unroll
        for (int e = 0; e < N; e++)
            if (v[e] == m) at = min(at, place(p.vec, base, lane, e));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
        s = (double)at;
    } else {
        const double md = (double)fmaxf(m, -kFltMax);
        double s1 = 0.0;
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            s += exp_neg((double)v[e] - md, p.rate, tab);
            s1 += exp_neg((double)v[e + 1] - md, p.rate, tab);
        }
        s = wave_sum_d(s + s1);
    }
    if (W > 1) {
        if (lane == 0) ss[wid] = s;
        __syncthreads();
        s = ss[0];
#pragma unroll
        for (int k = 1; k < W; k++) s = p.greedy ? fmin(s, ss[k]) : s + ss[k];
    }
    if (W == 1 ? lane == 0 : threadIdx.x == 0) {
        p.cmax[pos * p.nch + c] = m;
        p.csum[pos * p.nch + c] = s;
    }
}

// A row's verdict from its chunk statistics.
// The workgroup's waves take the positions in turn; the same sums in the same order wherever it is asked.  (Worked out again by every
// workgroup of the mass launch, which leaves it for the draw: a launch of its own for it would cost more.)
struct VerdictLds {
    double s[64];
    float m[64];
    int best[64], keep[64];
};

template <int NT> __device__ __forceinline__ Verdict verdict_of(const VerifyParams &p, int r, VerdictLds &L, const double (&tab)[32])
{
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int n = p.lens ? min(max(p.lens[r], 0), p.T) : p.T;
    for (int i = wid; i <= n; i += NT / 64) {
        const int64_t pos = (int64_t)r * (p.T + 1) + i;
        const int x = i < n ? p.drafts[(int64_t)r * p.T + i] : -1;
        const bool in = x >= 0 && x < p.vocab;
        const float lx = in ? p.logits[pos * p.ld + x] : 0.0f;
        const double qx = in && p.q ? (double)p.q[((int64_t)r * p.T + i) * p.q_ld + x] : 1.0;
        const double u = i < n ? (double)p.uniform[(int64_t)r * (p.T + 1) + i] : 0.0;
        float cm[kVerifyMaxChunks / 64], m = -INFINITY;
        double cs[kVerifyMaxChunks / 64];
#pragma unroll
        for (int k = 0; k < kVerifyMaxChunks / 64; k++) {
            const int c = k * 64 + lane;
            cm[k] = c < p.nch ? p.cmax[pos * p.nch + c] : -INFINITY;
            cs[k] = c < p.nch ? p.csum[pos * p.nch + c] : 0.0;
            m = fmaxf(m, cm[k]);
        }
        m = wave_max_f(m);
        const bool any = m > -INFINITY;
        double s = 0.0;
        int best = 0x7fffffff;
        if (p.greedy) {
#pragma unroll
            for (int k = 0; k < kVerifyMaxChunks / 64; k++)
                if (any && cm[k] == m) best = min(best, (int)cs[k]);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, 64));
        } else {
            // (no chunk with a finite maximum: every sum is 0)
#pragma unroll
            for (int k = 0; k < kVerifyMaxChunks / 64; k++)
                if (k * 64 < p.nch) s += cs[k] * exp_neg((double)fmaxf(cm[k], -kFltMax) - (double)fmaxf(m, -kFltMax), p.rate, tab);
            s = wave_sum_d(s);
        }
        if (lane == 0) {
            const double px = !in || !any ? 0.0 : p.greedy ? (x == best ? 1.0 : 0.0) : exp_neg((double)logit(lx) - (double)m, p.rate, tab) / s;
            L.keep[i] = in && any && u * qx < px;
            L.m[i] = m;
            L.s[i] = s;
            L.best[i] = any ? best : -1;
        }
    }
    __syncthreads();
    const unsigned long long refuse = __ballot(lane < n && !L.keep[lane < n ? lane : 0]);
    Verdict w;
    w.kept = refuse ? __ffsll((long long)refuse) - 1 : n;
    w.refused = refuse != 0;
    w.m = L.m[w.kept];
    w.s = L.s[w.kept];
    w.best = L.best[w.kept];
    return w;
}

// W waves a chunk, as above: four up to 12 chunks a CU (the whole verification of one row of 4 drafts 12.5 us, one wave a chunk 13.7; 32 rows
// 41.6 and 41.7; 64 rows 66.2 and 64.9)
template <int W> __global__ __launch_bounds__(VM) void k_verify_mass(const VerifyParams p)
{
    constexpr int N = VPL / W;
    __shared__ VerdictLds L;
    __shared__ double ss[VM / 64], tab[32];
    const int r = blockIdx.y, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int c = blockIdx.x * (VM / 64 / W) + wid / W, base = c * VC + wid % W * (VC / W);
    exp_table(kExp2[threadIdx.x & 31], tab);
    const Verdict w = verdict_of<VM>(p, r, L, tab);
    if (blockIdx.x == 0 && threadIdx.x == 0) p.verdicts[r] = w;          // (for the draw)
    if (!w.refused || !(w.s > 0.0) || (W == 1 && c >= p.nch)) return;
    const float *lrow = p.logits + ((int64_t)r * (p.T + 1) + w.kept) * p.ld, *qrow = p.q + ((int64_t)r * p.T + w.kept) * p.q_ld;
    float v[N], q[N];
    load_chunk<N>(lrow, base, lane, p.vocab, p.vec, -INFINITY, v);
    load_chunk<N>(qrow, base, lane, p.vocab, p.qvec && p.vec, 0.0f, q);
    if (p.vec && !p.qvec) {                                  // (the two rows have to be read in one order)
#pragma unroll
        for (int e = 0; e < N; e++) {
            const int j = place(1, base, lane, e);
            q[e] = j < p.vocab ? qrow[j] : 0.0f;
        }
    }
    const double inv_s = 1.0 / w.s;
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < N; e++)
        s += fmax(__builtin_fma(exp_neg((double)logit(v[e]) - (double)w.m, p.rate, tab), inv_s, -(double)q[e]), 0.0);
    s = wave_sum_d(s);
    if (W > 1) {
        if (lane == 0) ss[wid] = s;
        __syncthreads();
        if (wid % W) return;
#pragma unroll
        for (int k = 1; k < W; k++) s += ss[wid + k];
    }
    if (lane == 0 && c < p.nch) p.mass[(int64_t)r * p.nch + c] = s;
}

// inclusive sums over the workgroup's threads, in thread order, and the whole
__device__ __forceinline__ double block_scan(double v, double (&part)[VD / 64], double *all)
{
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    v = wave_scan_d(v);
    if (lane == 63) part[wid] = v;
    __syncthreads();
    double before = 0.0, a = 0.0;
#pragma unroll
    for (int w = 0; w < VD / 64; w++) {
        if (w == wid) before = a;
        a += part[w];
    }
    *all = a;
    return before + v;
}

__global__ __launch_bounds__(VD) void k_verify_draw(const VerifyParams p)
{
    __shared__ VerdictLds L;
    __shared__ double part[4][VD / 64], cut, tab[32];
    __shared__ int first[2], last[2];
    const int r = blockIdx.x, tid = threadIdx.x;
    constexpr int E = VC / VD;
    if (tid < 2) first[tid] = 0x7fffffff;
    if (tid < 2) last[tid] = -1;
    const double u = (double)p.uniform[(int64_t)r * (p.T + 1) + p.T];
    exp_table(kExp2[threadIdx.x & 31], tab);
    const Verdict w = p.verdicts ? p.verdicts[r] : verdict_of<VD>(p, r, L, tab);
    int token = -1;
    if (p.greedy) token = w.best;
    else if (w.s > 0.0) {
        const int64_t pos = (int64_t)r * (p.T + 1) + w.kept, qpos = (int64_t)r * p.T + w.kept;
        const float *row = p.logits + pos * p.ld, *qrow = p.q && w.refused ? p.q + qpos * p.q_ld : nullptr;
        // a looked-up draft that was refused: everything but itself is left over
        int x = w.refused && !p.q ? p.drafts[qpos] : -1;
        if (x >= p.vocab) x = -1;
        const double inv_s = 1.0 / w.s, md = (double)w.m;
        // a thread a chunk: mass of p (in units of the sum), and with a draft's distribution what p has over it
        const bool mine = tid < p.nch;
        const float cmx = mine ? p.cmax[pos * p.nch + tid] : -INFINITY;
        const double csm = mine ? p.csum[pos * p.nch + tid] : 0.0, left = mine && qrow ? p.mass[(int64_t)r * p.nch + tid] : 0.0;
        float xv[E];
        if (x >= 0) {                                         // the draft's own chunk, without it
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int j = x / VC * VC + e * VD + tid;
                xv[e] = j < p.vocab && j != x ? row[j] : -INFINITY;
            }
        }
        const double pm = csm * exp_neg((double)fmaxf(cmx, -kFltMax) - md, p.rate, tab);
        double cm = qrow ? left : pm, total;
        if (x >= 0) {
            double s = 0.0, without;
#pragma unroll
            for (int e = 0; e < E; e++) s += exp_neg((double)logit(xv[e]) - md, p.rate, tab);
            block_scan(s, part[3], &without);
            if (tid == x / VC) cm = without;
        }
        bool rest = qrow || x >= 0;
        double cum = block_scan(cm, part[0], &total);
        if (rest && !(total > 0.0)) {                         // nothing is left over: the token comes from p
            rest = false;
            cm = pm;
            cum = block_scan(cm, part[1], &total);
        }
        const double want = u * total;
        // (one LDS atomic a wave: one of every thread on one word cost 7 us.  A chunk without mass is never the one: the sums of neighbouring
        // lanes are associated differently, so its cum can lie a bit above its predecessor's)
        const int lane = tid & 63;
        const unsigned long long past = __ballot(mine && cm > 0.0 && cum > want);
        const unsigned long long with = __ballot(mine && cm > 0.0);
        if (past && lane == __ffsll((long long)past) - 1) atomicMin(&first[0], tid);
        if (with && lane == 63 - __clzll((long long)with)) atomicMax(&last[0], tid);
        __syncthreads();
        const int c = first[0] != 0x7fffffff ? first[0] : max(last[0], 0);     // (a number of 1 or more: the last chunk with any mass)
        // the chunk's tokens, E consecutive ones a thread
        const int j0 = c * VC + tid * E;
        float lv[E], qv[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            lv[e] = j0 + e < p.vocab ? row[j0 + e] : -INFINITY;
            qv[e] = rest && qrow && j0 + e < p.vocab ? qrow[j0 + e] : 0.0f;
        }
        if (tid == c) cut = cum - cm;
        double mass[E], sum = 0.0, all;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const double v = exp_neg((double)logit(lv[e]) - md, p.rate, tab);
            mass[e] = rest && qrow ? fmax(__builtin_fma(v, inv_s, -(double)qv[e]), 0.0) : rest && j0 + e == x ? 0.0 : v;
            sum += mass[e];
        }
        double upto = block_scan(sum, part[2], &all);
        upto += cut;                                          // (behind the scan's barrier: thread c has written it)
        int at = -1, lastj = -1;
        double a = upto - sum;
#pragma unroll
        for (int e = 0; e < E; e++) {
            a += mass[e];
            if (mass[e] > 0.0) {
                lastj = j0 + e;
                if (at < 0 && a > want) at = j0 + e;
            }
        }
        const unsigned long long hit = __ballot(at >= 0), some = __ballot(lastj >= 0);
        if (hit && lane == __ffsll((long long)hit) - 1) atomicMin(&first[1], at);
        if (some && lane == 63 - __clzll((long long)some)) atomicMax(&last[1], lastj);
        __syncthreads();
        token = first[1] != 0x7fffffff ? first[1] : last[1];  // (rounding past the chunk's end: its last token with any mass)
    }
    for (int i = tid; i <= p.T; i += VD)
        p.out_tokens[(int64_t)r * (p.T + 1) + i] = i < w.kept ? p.drafts[(int64_t)r * p.T + i] : i == w.kept ? token : -1;
    if (tid == 0) p.out_count[r] = w.kept + 1;
}

// A workgroup a row, half a wave a position: lane c holds candidate c.  The first refusal's remaining mass needs the draft's probability of
// each candidate, looked up in LDS.  64 rows of 4 drafts: 3.9 us, the latency of the launch and of three dependent loads.
__global__ __launch_bounds__(VT) void k_verify_topk(const int32_t *__restrict__ cand, const float *__restrict__ probs,
                                                    const int32_t *__restrict__ dcand, const float *__restrict__ dprobs,
                                                    const int32_t *__restrict__ drafts, const int32_t *__restrict__ lens,
                                                    const float *__restrict__ uniform, int T, int32_t *__restrict__ out_tokens,
                                                    int32_t *__restrict__ out_count)
{
    __shared__ int keep[64], sid[32];
    __shared__ float sp[32];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, c = tid & 31;
    const int n = lens ? min(max(lens[r], 0), T) : T;
    const float ud = uniform[r * (T + 1) + T];
    for (int i = tid >> 5; i < n; i += VT / 32) {
        const int x = drafts[r * T + i];
        const float u = uniform[r * (T + 1) + i];
        const int64_t at = (r * (T + 1) + i) * 32 + c, da = (r * T + i) * 32 + c;
        const int id = cand[at], did = dcand ? dcand[da] : -1;
        const float pv = probs[at], dv = dcand ? dprobs[da] : 0.0f;
        double px = id == x && pv > 0.0f ? (double)pv : 0.0, qx = dcand && did == x ? (double)dv : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            px += __shfl_xor(px, o, 32);
            qx += __shfl_xor(qx, o, 32);
        }
        if (c == 0) keep[i] = (double)u * (dcand ? qx : 1.0) < px;
    }
    __syncthreads();
    const unsigned long long refuse = __ballot(lane < n && !keep[lane < n ? lane : 0]);
    const int kept = refuse ? __ffsll((long long)refuse) - 1 : n;
    const int64_t at = (r * (T + 1) + kept) * 32 + c, da = (r * T + kept) * 32 + c;
    if (refuse && dcand && tid < 32) {
        sid[c] = dcand[da];
        sp[c] = dprobs[da];
    }
    const int id = cand[at];
    const float pv = probs[at];
    const double p = pv > 0.0f ? (double)pv : 0.0;
    __syncthreads();
    double w = p;
    if (refuse) {
        double q = 0.0;
        if (dcand) {
#pragma unroll
            for (int k = 0; k < 32; k++) q += sid[k] == id ? (double)sp[k] : 0.0;
        } else
            q = id == drafts[r * T + kept] ? 1.0 : 0.0;
        const double rest = fmax(p - q, 0.0);
        if (__any(rest > 0.0)) w = rest;
    }
    // cumulated in the candidates' order (both halves of a wave hold the same)
    double cum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double b = __shfl_up(cum, o, 32);
        if (c >= o) cum += b;
    }
    const double total = __shfl(cum, 31, 32);
    const unsigned hit = (unsigned)__ballot(w > 0.0 && cum > (double)ud * total), some = (unsigned)__ballot(w > 0.0);
    const int k = hit ? __ffs((int)hit) - 1 : some ? 31 - __clz((int)some) : -1;
    const int tok = __shfl(id, k < 0 ? 0 : k, 32), token = k < 0 ? -1 : tok;
    for (int i = tid; i <= T; i += VT) out_tokens[r * (T + 1) + i] = i < kept ? drafts[r * T + i] : i == kept ? token : -1;
    if (tid == 0) out_count[r] = kept + 1;
}

}  // namespace ifh

using namespace ifh;

static int64_t verify_chunks(int vocab) { return ((int64_t)vocab + VC - 1) / VC; }

extern "C" int64_t ifh_verify_drafts_ws_bytes(int nrows, int ndraft)
{
    if (nrows <= 0 || ndraft < 0 || ndraft > 63) return 0;
    return (int64_t)nrows * (kVerifyMaxChunks * ((ndraft + 1) * 12 + 8) + (int64_t)sizeof(Verdict));
}

extern "C" int ifh_verify_drafts_f32(const ifh_verify_desc *d, ifh_stream_t stream)
{
    IFH_CHECK_ARG(d && d->nrows >= 0);
    if (d->nrows == 0) return IFH_OK;
    IFH_CHECK_ARG(d->ndraft >= 0 && d->ndraft <= 63 && d->vocab >= 1 && verify_chunks(d->vocab) <= kVerifyMaxChunks);
    IFH_CHECK_ARG(d->logits && d->uniform && d->out_tokens && d->out_count && d->ws && (d->drafts || d->ndraft == 0));
    IFH_CHECK_ARG(d->ld >= d->vocab && (!d->draft_probs || d->q_ld >= d->vocab));
    IFH_CHECK_ARG(d->temperature >= 0.0 && d->temperature <= 1e6 && (d->temperature == 0.0 || d->temperature >= 1e-6));
    const int64_t positions = (int64_t)d->nrows * (d->ndraft + 1);
    IFH_CHECK_ARG(d->nrows < 65536 && positions < 65536);
    IFH_CHECK_ARG((((uintptr_t)d->ws) & 15) == 0 && d->ws_bytes >= ifh_verify_drafts_ws_bytes(d->nrows, d->ndraft));
    VerifyParams p = {};
    p.logits = d->logits; p.ld = d->ld; p.q = d->draft_probs; p.q_ld = d->q_ld;
    p.drafts = d->drafts; p.lens = d->lens; p.uniform = d->uniform;
    p.out_tokens = d->out_tokens; p.out_count = d->out_count;
    p.vocab = d->vocab; p.T = d->ndraft; p.nch = (int)verify_chunks(d->vocab);
    p.greedy = d->temperature == 0.0;
    p.rate.rate = 46.166241308446828 / (p.greedy ? 1.0 : d->temperature);
    p.rate.least = -40000.0 / p.rate.rate;
    p.vec = (((uintptr_t)d->logits) & 15) == 0 && d->ld % 4 == 0;
    p.qvec = (((uintptr_t)d->draft_probs) & 15) == 0 && d->q_ld % 4 == 0;
    const bool mass = !p.greedy && p.q && p.T > 0;
    p.verdicts = mass ? (Verdict *)d->ws : nullptr;
    p.csum = (double *)((Verdict *)d->ws + d->nrows);
    p.mass = p.csum + positions * p.nch;
    p.cmax = (float *)(p.mass + (int64_t)d->nrows * p.nch);
    hipStream_t st = as_stream(stream);
    if (positions * p.nch <= 32 * (int64_t)device_cu_count_physical())
        hipLaunchKernelGGL(k_verify_stats<4>, dim3((unsigned)p.nch, (unsigned)positions), dim3(VT), 0, st, p);
    else
        hipLaunchKernelGGL(k_verify_stats<1>, dim3((unsigned)(p.nch + 3) / 4, (unsigned)positions), dim3(VT), 0, st, p);
    IFH_LAUNCH_CHECK("verify stats");
    if (mass) {
        if ((int64_t)d->nrows * p.nch <= 12 * (int64_t)device_cu_count_physical())
            hipLaunchKernelGGL(k_verify_mass<4>, dim3((unsigned)(p.nch + VM / 256 - 1) / (VM / 256), (unsigned)d->nrows), dim3(VM), 0, st, p);
        else
            hipLaunchKernelGGL(k_verify_mass<1>, dim3((unsigned)(p.nch + VM / 64 - 1) / (VM / 64), (unsigned)d->nrows), dim3(VM), 0, st, p);
        IFH_LAUNCH_CHECK("verify mass");
    }
    hipLaunchKernelGGL(k_verify_draw, dim3((unsigned)d->nrows), dim3(VD), 0, st, p);
    IFH_LAUNCH_CHECK("verify draw");
    return IFH_OK;
}

extern "C" int ifh_verify_drafts_topk(const int32_t *cand, const float *probs, const int32_t *draft_cand, const float *draft_probs,
                                      const int32_t *drafts, const int32_t *lens, const float *uniform, int nrows, int ndraft,
                                      int32_t *out_tokens, int32_t *out_count, ifh_stream_t stream)
{
    IFH_CHECK_ARG(nrows >= 0);
    if (nrows == 0) return IFH_OK;
    IFH_CHECK_ARG(ndraft >= 0 && ndraft <= 63);
    IFH_CHECK_ARG(cand && probs && uniform && out_tokens && out_count && (drafts || ndraft == 0));
    IFH_CHECK_ARG((draft_cand == nullptr) == (draft_probs == nullptr));
    hipLaunchKernelGGL(k_verify_topk, dim3((unsigned)nrows), dim3(VT), 0, as_stream(stream), cand, probs, draft_cand, draft_probs, drafts, lens,
                       uniform, ndraft, out_tokens, out_count);
    IFH_LAUNCH_CHECK("verify topk");
    return IFH_OK;
}
