// Verification of drafted tokens (speculative decoding by rejection): ifh_verify_drafts_f32 on whole distributions,
// ifh_verify_drafts_topk on the top-k sampler's candidates.
//
// The draw compares a cumulated mass with a given number, and a vocabulary of 150 000 tokens has borders 1e-6 apart: masses are f64, so
// that neither the way a sum is split nor the exponential's rounding moves a border past the number (f32 exponentials would move one in
// every few hundred draws from a flat tail).  The f64 work (a short polynomial, ~20 operations a logit) stays under the time the logits
// take to arrive.
//   k_verify_stats   a chunk of a target row each: (max, sum of exp) of the chunk, or its arg-max for temperature 0
//   k_verify_mass    a chunk each: which draft the row refuses, and where one was, the mass of max(p - q, 0) in the chunk
//   k_verify_draw    a row each: the chunk and then the token where the cumulated mass passes the uniform number
#include "common.h"

namespace ifh {

constexpr int VC_THREADS = 256, VC_VEC = 8, VC = VC_THREADS * VC_VEC * 4;      // logits a chunk: 8192, 32 a thread

// e^x for x <= 0 in f64, relative error below 1e-12: x = k ln 2 + r, |r| <= ln 2 / 2, Taylor polynomial of degree 11 in r
__device__ __forceinline__ double exp_neg(double x)
{
    if (!(x > -700.0)) return 0.0;
    const double k = __builtin_rint(x * 1.4426950408889634);
    const double r = __builtin_fma(k, -1.9082149292705877e-10, __builtin_fma(k, -0.6931471803691238, x));
    double e = 2.505210838544172e-8;                       // 1 / 11!
    e = __builtin_fma(e, r, 2.755731922398589e-7);
    e = __builtin_fma(e, r, 2.7557319223985893e-6);
    e = __builtin_fma(e, r, 2.48015873015873e-5);
    e = __builtin_fma(e, r, 1.984126984126984e-4);
    e = __builtin_fma(e, r, 1.388888888888889e-3);
    e = __builtin_fma(e, r, 8.333333333333333e-3);
    e = __builtin_fma(e, r, 4.1666666666666664e-2);
    e = __builtin_fma(e, r, 0.16666666666666666);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    return __builtin_ldexp(e, (int)k);
}

// NaN counts as -inf; +inf as the largest finite value (its differences stay finite)
__device__ __forceinline__ float logit(float l) { return l == l ? fminf(l, 3.402823466e38f) : -INFINITY; }

struct VerifyParams {
    const float *logits;
    int64_t ld;
    const float *q;
    int64_t q_ld;
    const int32_t *drafts, *lens;
    const float *uniform;
    int32_t *out_tokens, *out_count;
    int vocab, nrows, T, nch;
    double inv_temp;
    int greedy, vec, qvec;
    float *cmax;                 // [rows * (T+1)][nch] chunk maxima
    double *csum;                // [rows * (T+1)][nch] chunk sums of exp((l - cmax) / temperature); greedy: the arg-max of the chunk
    double *mass;                // [rows][nch]
};

__device__ __forceinline__ void load_chunk(const float *row, int base, int vocab, int vec, float fill, float (&v)[VC_VEC * 4])
{
#pragma unroll
    for (int u = 0; u < VC_VEC; u++) {
        const int j = base + (u * VC_THREADS + (int)threadIdx.x) * 4;
        if (vec && j + 3 < vocab) {
            const float4 f = *reinterpret_cast<const float4 *>(row + j);
            v[4 * u] = f.x; v[4 * u + 1] = f.y; v[4 * u + 2] = f.z; v[4 * u + 3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * u + e] = j + e < vocab ? row[j + e] : fill;
        }
    }
}

__device__ __forceinline__ double wave_sum_d(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__global__ __launch_bounds__(VC_THREADS) void k_verify_stats(const VerifyParams p)
{
    __shared__ float sm[4];
    __shared__ double sd[4];
    const int64_t pos = blockIdx.y;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, base = blockIdx.x * VC;
    float v[VC_VEC * 4];
    load_chunk(p.logits + pos * p.ld, base, p.vocab, p.vec, -INFINITY, v);
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < VC_VEC * 4; e++) {
        v[e] = logit(v[e]);
        m = fmaxf(m, v[e]);
    }
    m = wave_max(m);
    if (lane == 0) sm[wid] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    double s = 0.0;
    if (p.greedy) {
        int at = 0x7fffffff;                                 // the first place of the maximum
#pragma unroll
        for (int e = VC_VEC * 4 - 1; e >= 0; e--)
            if (v[e] == m) at = base + ((e >> 2) * VC_THREADS + (int)threadIdx.x) * 4 + (e & 3);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
        s = (double)at;
        if (lane == 0) sd[wid] = s;
        __syncthreads();
        s = fmin(fmin(sd[0], sd[1]), fmin(sd[2], sd[3]));
    } else {
        const double md = (double)fmaxf(m, -3.402823466e38f);
#pragma unroll
        for (int e = 0; e < VC_VEC * 4; e++) s += exp_neg(((double)v[e] - md) * p.inv_temp);
        s = wave_sum_d(s);
        if (lane == 0) sd[wid] = s;
        __syncthreads();
        s = (sd[0] + sd[1]) + (sd[2] + sd[3]);
    }
    if (threadIdx.x == 0) {
        p.cmax[pos * p.nch + blockIdx.x] = m;
        p.csum[pos * p.nch + blockIdx.x] = s;
    }
}

// what a row's chunk statistics say: the number of drafts it keeps, whether the next one was refused, and the statistics of the
// position that is drawn.  One wave; the same sums in the same order in every workgroup that asks.
struct Verdict {
    int kept, refused, best;
    float m;
    double s;
};

__device__ __forceinline__ Verdict verdict_of(const VerifyParams &p, int r)
{
    const int lane = threadIdx.x & 63;
    Verdict w = {0, 0, -1, 0.0f, 0.0};
    const int n = p.lens ? min(max(p.lens[r], 0), p.T) : p.T;
    for (int i = 0; i <= n; i++) {
        const int64_t pos = (int64_t)r * (p.T + 1) + i;
        float m = -INFINITY;
        for (int c = lane; c < p.nch; c += 64) m = fmaxf(m, p.cmax[pos * p.nch + c]);
        m = wave_max(m);
        const bool any = m > -INFINITY;
        double s = 0.0;
        int best = 0x7fffffff;
        if (p.greedy) {
            for (int c = lane; c < p.nch; c += 64)
                if (any && p.cmax[pos * p.nch + c] == m) best = min(best, (int)p.csum[pos * p.nch + c]);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, 64));
        } else {
            for (int c = lane; c < p.nch; c += 64)
                s += p.csum[pos * p.nch + c] * exp_neg(((double)fmaxf(p.cmax[pos * p.nch + c], -3.402823466e38f) - (double)fmaxf(m, -3.402823466e38f)) * p.inv_temp);
            s = wave_sum_d(s);
        }
        w.kept = i;
        w.m = m;
        w.s = s;
        w.best = any ? best : -1;
        if (i == n) break;
        const int x = p.drafts[(int64_t)r * p.T + i];
        bool keep = false;
        if (x >= 0 && x < p.vocab && any) {
            const double qx = p.q ? (double)p.q[((int64_t)r * p.T + i) * p.q_ld + x] : 1.0;
            const double px = p.greedy ? (x == best ? 1.0 : 0.0) : exp_neg(((double)logit(p.logits[pos * p.ld + x]) - (double)m) * p.inv_temp) / s;
            keep = (double)p.uniform[(int64_t)r * (p.T + 1) + i] * qx < px;
        }
        if (!keep) {
            w.refused = 1;
            break;
        }
    }
    return w;
}

// mass of token j at the drawn position: max(p - q, 0) at a refused draft, else p (in units of the sum: the draw is relative)
__device__ __forceinline__ double rest_of(double e, double inv_s, bool has_q, float qv, bool is_draft)
{
    if (has_q) return fmax(e * inv_s - (double)qv, 0.0);
    return is_draft ? fmax(e * inv_s - 1.0, 0.0) : e * inv_s;
}

__global__ __launch_bounds__(VC_THREADS) void k_verify_mass(const VerifyParams p)
{
    __shared__ double sd[4];
    const int r = blockIdx.y, lane = threadIdx.x & 63, wid = threadIdx.x >> 6, base = blockIdx.x * VC;
    const Verdict w = verdict_of(p, r);
    if (p.greedy || !w.refused || !(w.s > 0.0)) return;
    float v[VC_VEC * 4], q[VC_VEC * 4];
    load_chunk(p.logits + ((int64_t)r * (p.T + 1) + w.kept) * p.ld, base, p.vocab, p.vec, -INFINITY, v);
    if (p.q) load_chunk(p.q + ((int64_t)r * p.T + w.kept) * p.q_ld, base, p.vocab, p.qvec, 0.0f, q);
    const int x = p.drafts[(int64_t)r * p.T + w.kept];
    const double inv_s = 1.0 / w.s;
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < VC_VEC * 4; e++) {
        const int j = base + ((e >> 2) * VC_THREADS + (int)threadIdx.x) * 4 + (e & 3);
        s += rest_of(exp_neg(((double)logit(v[e]) - (double)w.m) * p.inv_temp), inv_s, p.q != nullptr, p.q ? q[e] : 0.0f, j == x);
    }
    s = wave_sum_d(s);
    if (lane == 0) sd[wid] = s;
    __syncthreads();
    if (threadIdx.x == 0) p.mass[(int64_t)r * p.nch + blockIdx.x] = (sd[0] + sd[1]) + (sd[2] + sd[3]);
}

__global__ __launch_bounds__(VC_THREADS) void k_verify_draw(const VerifyParams p)
{
    __shared__ double part[VC_THREADS];
    __shared__ int found, last;
    const int r = blockIdx.x, tid = threadIdx.x;
    const Verdict w = verdict_of(p, r);
    int token = -1;
    if (p.greedy) token = w.best;
    else if (w.s > 0.0) {
        const int64_t pos = (int64_t)r * (p.T + 1) + w.kept;
        // the chunks' masses in order, the same in every thread
        bool rest = w.refused;
        double total = 0.0;
        if (rest) {
            for (int c = 0; c < p.nch; c++) total += p.mass[(int64_t)r * p.nch + c];
            rest = total > 0.0;
        }
        auto chunk = [&](int c) {
            return rest ? p.mass[(int64_t)r * p.nch + c]
                        : p.csum[pos * p.nch + c] * exp_neg(((double)fmaxf(p.cmax[pos * p.nch + c], -3.402823466e38f) - (double)w.m) * p.inv_temp);
        };
        if (!rest) {
            total = 0.0;
            for (int c = 0; c < p.nch; c++) total += chunk(c);
        }
        const double want = (double)p.uniform[(int64_t)r * (p.T + 1) + p.T] * total;
        double before = 0.0;
        int c = 0, full = 0;
        double fbefore = 0.0;
        for (; c < p.nch; c++) {                              // the first chunk in which the mass passes; rounding past the end: the last with any
            const double m = chunk(c);
            if (before + m > want) break;
            if (m > 0.0) {
                full = c;
                fbefore = before;
            }
            before += m;
        }
        if (c == p.nch) {
            c = full;
            before = fbefore;
        }
        // inside the chunk: 32 consecutive tokens a thread
        const float *row = p.logits + pos * p.ld, *qrow = p.q && rest ? p.q + ((int64_t)r * p.T + w.kept) * p.q_ld : nullptr;
        const int x = rest ? p.drafts[(int64_t)r * p.T + w.kept] : -1, j0 = c * VC + tid * (VC_VEC * 4);
        const double inv_s = 1.0 / w.s;
        auto mass_at = [&](int j) {
            const double e = exp_neg(((double)logit(row[j]) - (double)w.m) * p.inv_temp);
            return rest ? rest_of(e, inv_s, qrow != nullptr, qrow ? qrow[j] : 0.0f, j == x) : e;
        };
        double mine = 0.0;
        int lastj = -1;
        for (int e = 0; e < VC_VEC * 4; e++)
            if (j0 + e < p.vocab) {
                const double m = mass_at(j0 + e);
                mine += m;
                if (m > 0.0) lastj = j0 + e;
            }
        part[tid] = mine;
        if (tid == 0) found = last = -1;
        __syncthreads();
        if (lastj >= 0) atomicMax(&last, lastj);
        double pre = before;
        for (int t = 0; t < tid; t++) pre += part[t];
        if (pre <= want && pre + mine > want) {
            double a = pre;
            int at = lastj;
            for (int e = 0; e < VC_VEC * 4; e++)
                if (j0 + e < p.vocab) {
                    a += mass_at(j0 + e);
                    if (a > want) {
                        at = j0 + e;
                        break;
                    }
                }
            found = at;
        }
        __syncthreads();
        token = found >= 0 ? found : last;
    }
    for (int i = tid; i <= p.T; i += VC_THREADS)
        p.out_tokens[(int64_t)r * (p.T + 1) + i] = i < w.kept ? p.drafts[(int64_t)r * p.T + i] : i == w.kept ? token : -1;
    if (tid == 0) p.out_count[r] = w.kept + 1;
}

// One wave a row: lane c holds the target's candidate c, and of the draft's candidates one a step comes round by broadcast.
__global__ __launch_bounds__(64) void k_verify_topk(const int32_t *__restrict__ cand, const float *__restrict__ probs,
                                                    const int32_t *__restrict__ dcand, const float *__restrict__ dprobs,
                                                    const int32_t *__restrict__ drafts, const int32_t *__restrict__ lens,
                                                    const float *__restrict__ uniform, int T, int32_t *__restrict__ out_tokens,
                                                    int32_t *__restrict__ out_count)
{
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x, c = lane & 31;
    const bool mine = lane < 32;
    const int n = lens ? min(max(lens[r], 0), T) : T;
    int kept = 0, token = -1;
    for (int i = 0; i <= n; i++) {
        const int64_t at = (r * (T + 1) + i) * 32 + c;
        const int id = cand[at];
        const float pv = probs[at];
        const double p = mine && pv > 0.0f ? (double)pv : 0.0;
        double w = p;
        if (i < n) {
            const int x = drafts[r * T + i];
            int did = -1;
            float dp = 0.0f;
            if (dcand) {
                const int64_t da = (r * T + i) * 32 + c;
                did = dcand[da];
                dp = dprobs[da];
            }
            double q = 0.0;                                            // the draft's probability of this lane's candidate
            if (dcand) {
                for (int k = 0; k < 32; k++) {
                    const int kid = __shfl(did, k, 64);
                    const float kp = __shfl(dp, k, 64);                // (by every lane: a lane that is switched off hands nothing out)
                    q += kid == id ? (double)kp : 0.0;
                }
            } else
                q = id == x ? 1.0 : 0.0;
            double px = id == x ? p : 0.0, qx = dcand ? (mine && did == x ? (double)dp : 0.0) : 0.0;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                px += __shfl_xor(px, o, 64);
                qx += __shfl_xor(qx, o, 64);
            }
            if (!dcand) qx = 1.0;
            if ((double)uniform[r * (T + 1) + i] * qx < px) {
                kept = i + 1;
                continue;
            }
            const double rest = mine ? fmax(p - q, 0.0) : 0.0;
            if (__any(rest > 0.0)) w = rest;
        }
        // cumulated in the candidates' order
        double cum = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double b = __shfl_up(cum, o, 64);
            if (lane >= o) cum += b;
        }
        const double total = __shfl(cum, 31, 64);
        unsigned long long hit = __ballot(mine && cum > (double)uniform[r * (T + 1) + T] * total), some = __ballot(w > 0.0);
        int k = -1;
        if (some) k = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
        const int tok = __shfl(id, k < 0 ? 0 : k, 64);
        token = k < 0 ? -1 : tok;
        break;
    }
    for (int i = lane; i <= T; i += 64) out_tokens[r * (T + 1) + i] = i < kept ? drafts[r * T + i] : i == kept ? token : -1;
    if (lane == 0) out_count[r] = kept + 1;
}

}  // namespace ifh

using namespace ifh;

static int64_t verify_chunks(int vocab) { return ((int64_t)vocab + VC - 1) / VC; }
constexpr int kVerifyMaxChunks = 64;             // 524 288 tokens

extern "C" int64_t ifh_verify_drafts_ws_bytes(int nrows, int ndraft)
{
    if (nrows <= 0 || ndraft < 0) return 0;
    return (int64_t)nrows * kVerifyMaxChunks * ((ndraft + 1) * 12 + 8);
}

extern "C" int ifh_verify_drafts_f32(const ifh_verify_desc *d, ifh_stream_t stream)
{
    IFH_CHECK_ARG(d && d->nrows >= 0);
    if (d->nrows == 0) return IFH_OK;
    IFH_CHECK_ARG(d->ndraft >= 0 && d->ndraft <= 63 && d->vocab >= 1 && verify_chunks(d->vocab) <= kVerifyMaxChunks);
    IFH_CHECK_ARG(d->logits && d->uniform && d->out_tokens && d->out_count && d->ws && (d->drafts || d->ndraft == 0));
    IFH_CHECK_ARG(d->ld >= d->vocab && (!d->draft_probs || d->q_ld >= d->vocab));
    IFH_CHECK_ARG(d->temperature >= 0.0f && d->temperature <= 1e6f && (d->temperature == 0.0f || d->temperature >= 1e-6f));
    const int64_t positions = (int64_t)d->nrows * (d->ndraft + 1);
    IFH_CHECK_ARG(d->nrows < 65536 && positions < 65536);
    IFH_CHECK_ARG((((uintptr_t)d->ws) & 15) == 0 && d->ws_bytes >= ifh_verify_drafts_ws_bytes(d->nrows, d->ndraft));
    VerifyParams p = {};
    p.logits = d->logits; p.ld = d->ld; p.q = d->draft_probs; p.q_ld = d->q_ld;
    p.drafts = d->drafts; p.lens = d->lens; p.uniform = d->uniform;
    p.out_tokens = d->out_tokens; p.out_count = d->out_count;
    p.vocab = d->vocab; p.nrows = d->nrows; p.T = d->ndraft; p.nch = (int)verify_chunks(d->vocab);
    p.greedy = d->temperature == 0.0f;
    p.inv_temp = p.greedy ? 1.0 : 1.0 / (double)d->temperature;
    p.vec = (((uintptr_t)d->logits) & 15) == 0 && d->ld % 4 == 0;
    p.qvec = (((uintptr_t)d->draft_probs) & 15) == 0 && d->q_ld % 4 == 0;
    p.csum = (double *)d->ws;
    p.mass = p.csum + positions * p.nch;
    p.cmax = (float *)(p.mass + (int64_t)d->nrows * p.nch);
    hipStream_t st = as_stream(stream);
    hipLaunchKernelGGL(k_verify_stats, dim3((unsigned)p.nch, (unsigned)positions), dim3(VC_THREADS), 0, st, p);
    IFH_LAUNCH_CHECK("verify stats");
    if (!p.greedy && p.T > 0) {
        hipLaunchKernelGGL(k_verify_mass, dim3((unsigned)p.nch, (unsigned)p.nrows), dim3(VC_THREADS), 0, st, p);
        IFH_LAUNCH_CHECK("verify mass");
    }
    hipLaunchKernelGGL(k_verify_draw, dim3((unsigned)p.nrows), dim3(VC_THREADS), 0, st, p);
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
    hipLaunchKernelGGL(k_verify_topk, dim3((unsigned)nrows), dim3(64), 0, as_stream(stream), cand, probs, draft_cand, draft_probs, drafts, lens,
                       uniform, ndraft, out_tokens, out_count);
    IFH_LAUNCH_CHECK("verify topk");
    return IFH_OK;
}
