// Language-model operators for prompts laid end to end and for decode steps that share a prefix (the serving forms next to llm.hip's
// padded batches; InfernLLMWorker, Cluster/InfernLLMWorker.py:60-119):
//   k_rope_packed    rotary embedding of q and k and the append of k | v to the cache rows, tokens of all sequences end to end.
//   k_attn_rows      softmax(scale q k^T) v of row blocks: a row is one (token, query head), the G heads of a kv head adjacent, so a
//                    K / V tile serves every head of the group and a block of rows covers few tokens (little work past the diagonal).
//   k_attn_join      joins the partial results of row blocks whose keys were split.
#include "common.h"

#include <type_traits>

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

namespace ifh {

// Last s of the n sequences with reached(s), or 0 (reached: up to some s, the same for the whole wave): the lanes probe 64 of them at a time,
// one round trip up to 64 sequences, two up to 4096.
template <typename F> __device__ __forceinline__ int last_reached(int n, F reached)
{
    const int lane = threadIdx.x & 63;
    int lo = 0, range = n;
    while (range > 1) {
        const int step = (range + 63) >> 6;
        const int cnt = __popcll(__ballot(lane * step < range && reached(lo + lane * step)));
        const int first = (cnt > 0 ? cnt - 1 : 0) * step;
        lo += first;
        range = min(step, range - first);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// One thread per (token, head slot, 8 pairs j .. j + 7 of the head): the arithmetic and the roundings of k_rope_append (llm.hip).
// Bound by memory: qkv read once, q and k | v written once (64 prompts of 12 / 2 heads of 128, 87 MB: 18.3 us = 4.7 TB/s, where a large
// copy reaches 4.9); the loads start before the sequence is looked up, whose chain would otherwise stand in front of them (+2 us).
__global__ __launch_bounds__(256) void k_rope_packed(const uint16_t *__restrict__ qkv, int64_t qkv_ld, uint16_t *__restrict__ q_out,
                                                     int64_t q_ld, const float *__restrict__ cs, int table_len,
                                                     uint16_t *__restrict__ cache, int64_t cache_bs, int64_t cache_ts,
                                                     const int32_t *__restrict__ cu, const int32_t *__restrict__ pos0,
                                                     const int32_t *__restrict__ slot0, int nseqs, int nh, int nkv, int hd, int max_pos,
                                                     int64_t total)
{
    const int64_t idx0 = (int64_t)blockIdx.x * 256 + threadIdx.x, idx = idx0 < total ? idx0 : total - 1;      // (whole waves: they search together)
    const int half = hd >> 1, groups = half >> 3, slots = nh + 2 * nkv;
    const int j = (int)(idx % groups) * 8, slot = (int)((idx / groups) % slots);
    const int i = (int)(idx / ((int64_t)groups * slots));
    const uint16_t *src = qkv + i * qkv_ld + (int64_t)slot * hd;
    const uint4 lo = *reinterpret_cast<const uint4 *>(src + j), hi = *reinterpret_cast<const uint4 *>(src + j + half);
    // the wave's first token's sequence; a later token's lies behind it
    const int i0 = __builtin_amdgcn_readfirstlane(i);
    int s = last_reached(nseqs, [&](int at) { return cu[at] <= i0; });
    if (cu[s + 1] <= i) {
        int hi_s = nseqs;
        while (s < hi_s) {
            const int mid = (s + hi_s) >> 1;
            if (cu[mid + 1] <= i) s = mid + 1; else hi_s = mid;
        }
    }
    if (idx0 >= total || s >= nseqs || i < cu[s]) return;
    const int t = i - cu[s], pos = pos0[s] + t, at = (slot0 ? slot0[s] : pos0[s]) + t;
    if (pos < 0 || pos >= table_len) return;
    if (slot >= nh && (at < 0 || at >= max_pos)) return;
    uint16_t *dst = slot < nh ? q_out + i * q_ld + (int64_t)slot * hd
                              : cache + (int64_t)s * cache_bs + (int64_t)at * cache_ts + (int64_t)(slot - nh) * hd;
    if (slot >= nh + nkv) {                 // value head: plain copy
        *reinterpret_cast<uint4 *>(dst + j) = lo;
        *reinterpret_cast<uint4 *>(dst + j + half) = hi;
        return;
    }
    const float *cp = cs + ((int64_t)pos * half + j) * 2;
    uint4 olo, ohi;
    const uint32_t *ul = reinterpret_cast<const uint32_t *>(&lo), *uh = reinterpret_cast<const uint32_t *>(&hi);
    uint32_t *pl = reinterpret_cast<uint32_t *>(&olo), *ph = reinterpret_cast<uint32_t *>(&ohi);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float4 c4 = *reinterpret_cast<const float4 *>(cp + 4 * e);       // cos, sin of pairs 2 e, 2 e + 1
        const float a0 = __uint_as_float(ul[e] << 16), a1 = __uint_as_float(ul[e] & 0xffff0000u);
        const float b0 = __uint_as_float(uh[e] << 16), b1 = __uint_as_float(uh[e] & 0xffff0000u);
        pl[e] = f32x2_to_bf16x2(a0 * c4.x - b0 * c4.y, a1 * c4.z - b1 * c4.w);
        ph[e] = f32x2_to_bf16x2(b0 * c4.x + a0 * c4.y, b1 * c4.z + a1 * c4.w);
    }
    *reinterpret_cast<uint4 *>(dst + j) = olo;
    *reinterpret_cast<uint4 *>(dst + j + half) = ohi;
}

// How the rows of a key set find their keys.
//   PACKED   sequence s has the tokens cu[s] .. cu[s+1]-1 and the first lim[s] keys of cache row s; its last token sees them all,
//            each earlier one a key less (causal, aligned at the end)
//   PREFIX   every token sees the first lim[token / T] keys (all of them without a list) of one shared row
//   OWN      token i of row b = i / T sees the first lim[i] keys of cache row b
enum { ROWS_PACKED, ROWS_PREFIX, ROWS_OWN };

// one kind of keys of a launch: `parts` parts of part_tiles tiles for each of `blocks` row blocks and each kv head
struct KeySet {
    const uint16_t *kv;
    int64_t bs, ts;
    const int32_t *lim;
    int mode, narrow, max_keys, blocks, parts, part_tiles;
    int part0;                             // the first part's place in the partial results
};

struct RowsParams {
    const uint16_t *q;
    int64_t q_ts;
    int v_off;
    uint16_t *out;
    int64_t o_ts;
    const int32_t *cu;
    int ntokens, nseqs, nkv, G, T;
    float scale;
    KeySet ks[2];
    int first, pairs;                      // workgroups of ks[0] (the others are ks[1]'s), and how many 256s of both are dealt in turn
    int joint;                             // ks[1]'s workgroups go through ks[0]'s keys themselves and write out
    // Partial results, or NULL: write out.  The rows of a kv head (token G + head of the group) in tiles of 32, a tile as the accumulators
    // hold it: part_o f32 [parts][nkv][row_tiles][hd / 4][32 rows][4], unnormalised; part_ml f32 [parts][nkv][row_tiles][32][2] (max, sum).
    int row_tiles;
    float *part_o, *part_ml;
};

enum { ROWS_MIXED, ROWS_LONG, ROWS_BOTH };
constexpr float kNoKeys = -3.402823466e38f;     // the maximum of a row that saw nothing: no score lies below
constexpr int kWideRows = 128, kNarrowRows = 32, kKeys = 32;

// max over lanes l and l ^ 32, every lane gets it
__device__ __forceinline__ float max_half(float m)
{
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const unsigned u = __float_as_uint(m);
    const u32x2 r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    float a;
    asm("v_max_f32 %0, %1, %2" : "=v"(a) : "v"(__uint_as_float(r.x)), "v"(__uint_as_float(r.y)));
    return a;
}

// the largest of a wave's values, in every lane (shifts within 16 lanes, then lane 15 of rows 0 and 2 and lane 31 handed on)
template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_max_i(int v)
{
    return max(v, __builtin_amdgcn_update_dpp((int)0x80000000, v, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ int wave_max_i(int v)
{
    v = dpp_max_i<0x111, 0xF>(v);
    v = dpp_max_i<0x112, 0xF>(v);
    v = dpp_max_i<0x114, 0xF>(v);
    v = dpp_max_i<0x118, 0xF>(v);
    v = dpp_max_i<0x142, 0xA>(v);
    v = dpp_max_i<0x143, 0xC>(v);
    return __builtin_amdgcn_readlane(v, 63);
}

// 16 bytes a lane from BASE + VOFF (a lane's offset) to LDS address DST + 16 lane
#define ROWS_DMA(VOFF, BASE, DST)                                                                                          \
    do {                                                                                                                   \
        unsigned keep_;                                                                                                    \
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0" \
                     : "=&s"(keep_) : "v"(VOFF), "s"(BASE), "s"(DST) : "memory");                                          \
    } while (0)

// The keys of a tile in LDS.  Rows are unpadded (the DMA writes 16 bytes a lane in a row), so the 16-byte chunks of key r are permuted on
// the source side: K chunk c at c ^ (r % 16) (head_dim 64: c ^ (r / 2 % 8)), so that the 16 keys a ds_read_b128 reads at once lie in 16
// different bank groups; V chunks in groups of four, group g at g ^ (r % 4) (head_dim 64: g ^ (r / 2 % 2)), so that the four keys x 64
// bytes of a transposed read do.
template <int HD> __device__ __forceinline__ int kperm(int r) { return HD == 128 ? r & 15 : (r >> 1) & 7; }
template <int HD> __device__ __forceinline__ int vperm(int r) { return HD == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }

// A wave's 32 rows: S^T = K Q^T and O^T = V^T P^T with the 32 x 32 x 16 MFMA.  A lane holds one row's scores of 16 of every 32 keys, so the
// softmax of a row is lane-local up to one exchange with lane ^ 32, and P goes from the accumulators of the first product into the operand
// of the second without leaving the lane (its 8 keys are 8 half + {0..3, 8..11} + 4 (lane / 32): V^T is read in that order, transposed by
// ds_read_b64_tr_b16).  Sums and maxima are f32.  The second product takes P as the sum of two bf16 (P16 false: P rounded, and what the
// rounding left, rounded: together within 2^-16 of P), so that the result has the bits of f32 probabilities; a caller may have the first
// alone (P16: within 2^-8, as the prompt kernel of llm.hip), which saves one of three products and the splitting.  Us a call, sum and
// rounded: one prompt of 8191 tokens, 40 / 8 heads of 128, 860 and 627; 64 prompts of 12 / 2 heads 35 and 31; 64 rows of 5 tokens behind
// 8001 shared keys 120 and 104, 64 single tokens behind 2048 15.0 and 14.4.
template <int HD, bool FEW, bool P16>
struct WaveRows {
    static constexpr int NS = HD / 16, ND = HD / 32, ROWB = HD * 2;
    bf16x8_t qf[NS];
    f32x16 o[ND];
    float ms, l;                     // about the running maximum, in the exponent (every lane of a row), and the sum (this lane's keys)
    float c1;                        // scale log2 e
    unsigned ka, va;                 // LDS offsets of this lane's first fragments in a tile: the others' differ in one bit field

    __device__ __forceinline__ void init(float scale, int lane)
    {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
        ms = 0.0f;
        l = 0.0f;
        c1 = scale * 1.4426950408889634f;
        const int l32 = lane & 31, h2 = lane >> 5;
        ka = (unsigned)(l32 * ROWB + (h2 ^ kperm<HD>(l32)) * 16);
        // lane i of a 16-lane group hands in key i / 4, columns 4 (i % 4) .. + 3 of a 4-key x 16-dim block and gets column i
        const int key = 4 * h2 + ((lane & 15) >> 2), c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        va = (unsigned)(key * ROWB + (c ^ vperm<HD>(key)) * 16 + (lane & 1) * 8);
    }
    __device__ __forceinline__ void load_q(const uint16_t *q, int h2)
    {
#pragma unroll
        for (int s = 0; s < NS; s++) qf[s] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const uint4 *>(q + 16 * s + 8 * h2));
    }
    // (before the first tile is waited for: left to hipcc the wait for q falls behind the next tile's DMA)
    __device__ __forceinline__ void wait_q()
    {
#pragma unroll
        for (int s = 0; s < NS; s++) asm volatile("" : : "v"(qf[s]));
    }
    // scores of the 32 keys of K tile kt, the fragments AHEAD products ahead; between(i) is called before product i
    template <typename F> __device__ __forceinline__ void scores(const unsigned char *lds, unsigned at, f32x16 &s, F between)
    {
        constexpr int AHEAD = 4;
        bf16x8_t kf[AHEAD];
        unsigned k0 = at + ka;
        if constexpr (FEW) asm volatile("" : "+v"(k0));         // (else hipcc keeps every fragment's address in a register)
        auto frag = [&](int i) { return *reinterpret_cast<const bf16x8_t *>(lds + (k0 ^ (32u * i))); };
        s = (f32x16){0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < AHEAD; i++) kf[i] = frag(i);
#pragma unroll
        for (int i = 0; i < NS; i++) {
            between(i);
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i % AHEAD], qf[i], s, 0, 0, 0);
            if (i + AHEAD < NS) kf[i % AHEAD] = frag(i + AHEAD);
        }
    }
    // scores -> unnormalised probabilities 2^(s c1 - ms); rel: keys of the tile this lane's row sees, minus 4 (lane / 32); first: set at the
    // wave's first tile of a range of keys.  ms starts as the maximum of the first tile that a row sees anything of (what it sees of a range
    // is its keys up to lim, so the range's first tile or none; first stays set while a row has seen keys, but no score above -inf) and is
    // raised only when a later tile exceeds it by more than 8 (a wave decides at once): p stays below 2^8, sums in f32 lose nothing by it,
    // and the rescaling of the accumulators is skipped for almost every tile.
    __device__ __forceinline__ void softmax(f32x16 &s, bool mask, int rel, bool &first)
    {
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = __builtin_fmaf(s[e], c1, -ms);
        if (mask) {
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = 8 * (e >> 2) + (e & 3) < rel ? s[e] : -INFINITY;
        }
        // (two chains: a maximum of three waits for the one before it)
        float mx = fmaxf(s[0], s[1]), my = fmaxf(s[2], s[3]);
#pragma unroll
        for (int e = 4; e < 16; e += 4) {
            mx = fmaxf(fmaxf(mx, s[e]), s[e + 1]);
            my = fmaxf(fmaxf(my, s[e + 2]), s[e + 3]);
        }
        mx = max_half(fmaxf(mx, my));
        if (first || __any(mx > 8.0f)) {
            const bool unset = first && l + __shfl_xor(l, 32, 64) == 0.0f;
            const bool none = unset && !(mx > -INFINITY);
            const float raise = none ? 0.0f : unset ? mx : fmaxf(mx, 0.0f);
            const float alpha = unset ? 1.0f : __builtin_amdgcn_exp2f(-raise);
            ms += raise;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= alpha;
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] -= raise;
            first = __any(none && rel > 0);
        }
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; e++) {
            s[e] = __builtin_amdgcn_exp2f(s[e]);
            ls[e & 3] += s[e];
        }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    }
    // the sum over both lanes of a row; a row that saw nothing counts for nothing in a join
    __device__ __forceinline__ void finish()
    {
        l += __shfl_xor(l, 32, 64);
        ms = l > 0.0f ? ms : kNoKeys;
    }
    // O^T += V^T P^T, V tile vt; v: the fragments of its first 16 keys, read before the softmax
    __device__ __forceinline__ void values(const unsigned char *lds, unsigned at, int kk, bf16x8_t (&v)[ND])
    {
        typedef __attribute__((address_space(3))) bf16x4_t *lds4;
        unsigned v0 = at + va;
        if constexpr (FEW) asm volatile("" : "+v"(v0));
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const bf16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(lds + (v0 ^ (64u * d)) + kk * 16 * ROWB));
            const bf16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(lds + (v0 ^ (64u * d)) + (kk * 16 + 8) * ROWB));
            v[d] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // the second half of two probabilities whose roundings are `hi`
    static __device__ __forceinline__ uint32_t rest(float a, float b, uint32_t hi)
    {
        return f32x2_to_bf16x2(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
    }
    __device__ __forceinline__ void accumulate(const unsigned char *lds, unsigned at, const f32x16 &s, bf16x8_t (&v)[ND])
    {
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            const int e0 = kk * 8;
            bf16x8_t next[ND];
            if (kk == 0) values(lds, at, 1, next);
            uint4 pb;
            pb.x = f32x2_to_bf16x2(s[e0], s[e0 + 1]);
            pb.y = f32x2_to_bf16x2(s[e0 + 2], s[e0 + 3]);
            pb.z = f32x2_to_bf16x2(s[e0 + 4], s[e0 + 5]);
            pb.w = f32x2_to_bf16x2(s[e0 + 6], s[e0 + 7]);
            const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, pb);
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[d], pf, o[d], 0, 0, 0);
            if constexpr (!P16) {
                const uint4 lo = make_uint4(rest(s[e0], s[e0 + 1], pb.x), rest(s[e0 + 2], s[e0 + 3], pb.y), rest(s[e0 + 4], s[e0 + 5], pb.z),
                                            rest(s[e0 + 6], s[e0 + 7], pb.w));
                const bf16x8_t pl = __builtin_bit_cast(bf16x8_t, lo);
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[d], pl, o[d], 0, 0, 0);
            }
            if (kk == 0) {
#pragma unroll
                for (int d = 0; d < ND; d++) v[d] = next[d];
            }
        }
    }
};

// Four waves.  Two forms of a workgroup, by KeySet::narrow:
//   wide    128 rows, a wave 32 of them.  K / V tiles of 32 keys come by LDS-DMA into a ring of buffers, the next tile (ROWS_BOTH: the next
//           two) in flight while this one is multiplied, one barrier a tile.
//   narrow  32 rows, shared by the waves: a wave takes every fourth tile of 32 keys, by itself (its own K and V buffer, the next K in flight
//           from the end of the first product on, no barrier), and the four results are joined in LDS.  For the few rows of a decode step,
//           whose work is bringing the keys: 128 rows would leave three waves idle.
// and three instances of the kernel:
//   ROWS_LONG    every workgroup is wide and its rows packed.  Three workgroups a CU (162 registers, 32 KB).  Bound by the matrix unit and
//                the vector unit in turn, at the clock that the power budget leaves (a tile of a wave: 768 clocks of products, ~550 of
//                softmax and splitting; 512 and ~400 with rounded probabilities): one prompt of 8191 tokens, 40 / 8 heads of 128,
//                850-865 us = 0.8 PFLOP/s of the formula, 1.2 of the matrix unit (rounded 625-655 us, 1.05-1.10 of both).
//   ROWS_MIXED   either form, decided at run time.  Two workgroups a CU (narrow: 68 KB, for four waves' buffers and results).  Bound by the
//                latency of a few dependent loads: a step of 64 rows behind 2048 shared keys 11.3 us + 4 us for the join.
//   ROWS_BOTH    wide and narrow ones that share a CU, where both key sets fill the device: two that multiply beside one that waits for
//                memory.  A narrow workgroup has three waves with keys, so that three workgroups fit a CU's LDS, and fragment addresses are
//                worked out again for every tile (two registers instead of twelve, so that three fit its registers).  Beside the other
//                key set's traffic a tile takes longer to come than to multiply, so wide ones bring two ahead.  64 rows of 5 tokens behind
//                8001 keys, 40 / 8 heads: 112 us (ROWS_MIXED 129); 48 rows of 4 behind 16000 118 us (132); 64 rows of 3 behind 4000, 14 / 2
//                heads of 64, 21.5 us (22.7).  In the other two neither pays (ROWS_LONG with both: 1 % slower, ROWS_MIXED 2 %).
template <int HD, int FORM, bool P16>
__global__ __launch_bounds__(256, FORM == ROWS_MIXED ? 2 : 3) void k_attn_rows(const RowsParams p)
{
    constexpr bool LONG = FORM == ROWS_LONG;
    constexpr int ROWB = HD * 2, ND = HD / 32, NW = FORM == ROWS_BOTH ? 3 : 4, RING = FORM == ROWS_BOTH ? 3 : 2;
    constexpr int CH = HD / 8, PK = 1024 / ROWB;               // chunks of a key, keys of a DMA instruction
    constexpr int TILE = kKeys * ROWB;
    constexpr int JROW = HD * 4 + 16, JWAVE = 32 * JROW;        // narrow: a wave's result in LDS, rows padded by one chunk
    constexpr int BYTES = LONG ? 2 * RING * TILE : 2 * NW * TILE > NW * (JWAVE + 256) ? 2 * NW * TILE : NW * (JWAVE + 256);
    __shared__ __attribute__((aligned(1024))) unsigned char lds[BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, h2 = lane >> 5;
    // Two key sets: 256 workgroups of one, 256 of the other, so that a CU holds one that multiplies (a part of the prefix) beside one that
    // waits for memory (own keys), then what is left of either.
    bool second = false;
    int wg = blockIdx.x;
    if (FORM == ROWS_MIXED && p.joint) second = true;
    else if (!LONG) {
        const int blk = wg >> 8;
        if (blk < 2 * p.pairs) {
            second = blk & 1;
            wg = (blk >> 1) * 256 + (wg & 255);
        } else {
            wg -= p.pairs * 256;
            second = wg >= p.first;
            wg -= second ? p.first - p.pairs * 256 : 0;
        }
    }
    const KeySet &ks = p.ks[second ? 1 : 0];
    const bool narrow = !LONG && ks.narrow;
    const int mode = LONG ? ROWS_PACKED : ks.mode, id = wg;
    // kv head, row block, part: neighbours on different XCDs, so that with 2, 4 or 8 kv heads an XCD's L2 holds its own heads' keys
    const int G = p.G, kvh = id % p.nkv, bp = id / p.nkv, part = bp / ks.blocks;
    const int rs = narrow ? 5 : 7, R = 1 << rs;                // rows of a block
    static_assert(kNarrowRows == 1 << 5 && kWideRows == 1 << 7, "rows of a block");
    int xb = bp - part * ks.blocks;

    // the block's sequence: tokens [n0, n1), first row of the block within it, its cache row and the keys it may read
    int n0, n1, row0, kbatch, klen;
    if (mode == ROWS_PACKED) {
        // sequence s owns the block slots floor(cu[s] G / R) + s .. : at least ceil(len G / R) of them, so no table of blocks is needed;
        // the last blocks of a long prompt see the most keys and start first
        xb = ks.blocks - 1 - xb;
        const int lo = last_reached(p.nseqs, [&](int at) { return (int)(((int64_t)p.cu[at] * G) >> rs) + at <= xb; });
        n0 = min(max(p.cu[lo], 0), p.ntokens);
        n1 = min(max(p.cu[lo + 1], n0), p.ntokens);
        const int blk = xb - ((int)(((int64_t)n0 * G) >> rs) + lo);
        if (blk < 0 || (int64_t)blk * R >= (int64_t)(n1 - n0) * G) return;
        row0 = blk * R;
        kbatch = lo;
        klen = min(max(ks.lim[lo], 0), ks.max_keys);
    } else if (mode == ROWS_PREFIX) {
        n0 = 0;
        n1 = p.ntokens;
        row0 = xb * R;
        kbatch = 0;
        klen = ks.max_keys;
    } else {
        const int blocks = (p.T * G + R - 1) / R;
        kbatch = xb / blocks;
        n0 = kbatch * p.T;
        n1 = n0 + p.T;
        row0 = (xb - kbatch * blocks) * R;
        klen = ks.max_keys;
    }
    const int n = n1 - n0, w0 = row0 + (narrow ? 0 : wid * 32), row = w0 + l32, t = row / G, g = row - t * G;
    const bool ok = t < n;
    const int tok = n0 + (ok ? t : 0), head = kvh * G + (ok ? g : 0);
    WaveRows<HD, FORM == ROWS_BOTH, P16> w;
    w.load_q(p.q + (int64_t)tok * p.q_ts + (int64_t)head * HD, h2);       // in flight while the limits are looked up
    int lim, wmax, wmin, kmax;                                 // keys this lane's row sees; most and fewest of the wave's rows; most of the block's
    if (mode == ROWS_PACKED) {
        const int past = klen - n + 1;
        lim = ok ? max(past + t, 0) : 0;
        wmax = w0 / G < n ? max(past + min((w0 + 31) / G, n - 1), 0) : 0;
        wmin = max(past + min(w0 / G, n - 1), 0);
        kmax = max(past + min((row0 + R - 1) / G, n - 1), 0);
    } else {
        lim = !ok ? 0 : !ks.lim ? klen : min(max(ks.lim[mode == ROWS_PREFIX ? tok / p.T : tok], 0), klen);
        wmax = wave_max_i(lim);
        wmin = -wave_max_i(ok ? -lim : -klen);
        kmax = wmax;
        if (!narrow) {
            int *smax = reinterpret_cast<int *>(lds);
            if (lane == 0) smax[wid] = wmax;
            __syncthreads();
            kmax = max(max(smax[0], smax[1]), max(smax[2], smax[3]));
            __syncthreads();
        }
    }
    wmax = __builtin_amdgcn_readfirstlane(wmax);
    wmin = __builtin_amdgcn_readfirstlane(wmin);
    kmax = __builtin_amdgcn_readfirstlane(kmax);
    int kt0 = 0, kt1 = (kmax + kKeys - 1) / kKeys;
    if (p.part_o) {
        kt0 = part * ks.part_tiles;
        kt1 = min(kt1, kt0 + ks.part_tiles);
    }

    w.init(p.scale, lane);
    const unsigned lbase = (unsigned)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)lds);
    unsigned ts2 = (unsigned)ks.ts * 2u;
    const unsigned char *ksrc = reinterpret_cast<const unsigned char *>(ks.kv + (int64_t)kbatch * ks.bs + (int64_t)kvh * HD);
    const unsigned char *vsrc = ksrc + (int64_t)p.v_off * 2;
    const int64_t pt = ((int64_t)(ks.part0 + part) * p.nkv + kvh) * p.row_tiles;        // first tile of this part and kv head

    if (!narrow) {
        // DMA: piece j of wave w brings keys (4 j + w) PK .. + PK - 1 of the tile (the permutation of a chunk is the same in every piece);
        // lane l -> key l / CH of the piece, LDS chunk l % CH.  The pieces of the next tile go out one by one between the products of this
        // one's scores: eight in a row hold a wave up for 500 clocks, with the matrix unit idle.
        constexpr int PIECES = TILE / 4096;
        const int drow = wid * PK + lane / CH, dpos = lane % CH;
        const unsigned kch = (unsigned)(dpos ^ kperm<HD>(drow)) * 16u, vch = (unsigned)(dpos ^ vperm<HD>(drow)) * 16u;
        unsigned ro[PIECES];
#pragma unroll
        for (int j = 0; j < PIECES; j++) ro[j] = (unsigned)(drow + j * 4 * PK) * ts2;
        // piece j of K (j < PIECES) or V of tile kt; past the end of the block's keys: the last key again, masked below
        auto piece = [&](int kt, unsigned at, int j) {
            const bool v = j >= PIECES;
            const int jj = v ? j - PIECES : j;
            const unsigned end = (unsigned)min(kmax - 1 - kt * kKeys, kKeys - 1) * ts2;
            const unsigned dst = lbase + at + (unsigned)wid * 1024u + (unsigned)((v ? TILE : 0) + jj * 4096);
            ROWS_DMA(min(ro[jj], end) + (v ? vch : kch), (v ? vsrc : ksrc) + (int64_t)kt * kKeys * (int64_t)ts2, dst);
        };
        auto whole = [&](int kt, unsigned at) {
#pragma unroll
            for (int j = 0; j < 2 * PIECES; j++) piece(kt, at, j);
        };
        if (kt0 < kt1) whole(kt0, 0);
        if (RING == 3 && kt0 + 1 < kt1) whole(kt0 + 1, 2 * TILE);
        w.wait_q();
        // the tile has landed (the next one may still be on its way), and the buffer before it is no longer read
        auto landed = [&](bool next) {
            if (RING == 2 || !next) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            else if (PIECES == 2) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
            __syncthreads();
        };
        unsigned at = 0, far = (RING - 1) * 2 * TILE;          // buffers of this tile and of the one that is brought meanwhile
        auto on = [&]() {
            at = at == (RING - 1) * 2 * TILE ? 0 : at + 2 * TILE;
            far = far == (RING - 1) * 2 * TILE ? 0 : far + 2 * TILE;
        };
        bool first = true;
        auto tile = [&](int kt, auto more) {
            const int kbase = kt * kKeys;
            f32x16 s;
            w.scores(lds, at, s, [&](int i) {
                if constexpr (decltype(more)::value)
                    if (i % 2 == 0) piece(kt + RING - 1, far, i / 2);
            });
            bf16x8_t v[ND];
            w.values(lds, at + TILE, 0, v);
            w.softmax(s, kbase + kKeys > wmin, lim - kbase - 4 * h2, first);
            w.accumulate(lds, at + TILE, s, v);
            on();
        };
        if (wmax == 0)                                         // a wave without rows, or whose rows see nothing: brings its pieces only
            for (int kt = kt0; kt < kt1; kt++) {
                landed(kt + 1 < kt1);
                if (kt + RING - 1 < kt1) whole(kt + RING - 1, far);
                on();
            }
        else {
            int kt = kt0;
            for (; kt + RING - 1 < kt1; kt++) {
                landed(true);
                tile(kt, std::true_type{});
            }
            for (; kt < kt1; kt++) {
                landed(kt + 1 < kt1);
                tile(kt, std::false_type{});
            }
        }
        w.finish();
        if (p.part_o) {
            if (!ok) return;
            const int r = tok * G + g;
            const int64_t at = (pt + (r >> 5)) * 32 + (r & 31);
            if (h2 == 0) *reinterpret_cast<float2 *>(p.part_ml + at * 2) = make_float2(w.ms, w.l);
            float *po = p.part_o + (pt + (r >> 5)) * (32 * HD) + ((r & 31) + 32 * h2) * 4;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4 *>(po + (8 * d + e / 2) * 128) = make_float4(w.o[d][e], w.o[d][e + 1], w.o[d][e + 2], w.o[d][e + 3]);
            return;
        }
        // A lane holds dims 8 i + 4 (lane / 32) .. + 3 of its row: halves of neighbouring groups of eight are exchanged with lane ^ 32, so
        // that a lane stores whole groups (16 bytes of bf16) and a row's two lanes 32 bytes in a row.  (Whole rows by way of LDS: no gain.)
        const float inv = w.l > 0.0f ? 1.0f / w.l : 0.0f;
        uint16_t *op = p.out + (int64_t)tok * p.o_ts + (int64_t)head * HD + 8 * h2;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
                const u32x2 x = __builtin_amdgcn_permlane32_swap(f32x2_to_bf16x2(w.o[d][e] * inv, w.o[d][e + 1] * inv),
                                                                 f32x2_to_bf16x2(w.o[d][e + 4] * inv, w.o[d][e + 5] * inv), false, false);
                const u32x2 y = __builtin_amdgcn_permlane32_swap(f32x2_to_bf16x2(w.o[d][e + 2] * inv, w.o[d][e + 3] * inv),
                                                                 f32x2_to_bf16x2(w.o[d][e + 6] * inv, w.o[d][e + 7] * inv), false, false);
                if (ok) *reinterpret_cast<uint4 *>(op + 32 * d + 2 * e) = make_uint4(x.x, y.x, x.y, y.y);
            }
        return;
    }

    // narrow: piece j brings keys j PK .. + PK - 1 of the wave's tile
    constexpr int PIECES = TILE / 1024;
    const unsigned kdst = lbase + (unsigned)wid * (2 * TILE), vdst = kdst + TILE;
    const int drow = lane / CH, dpos = lane % CH;
    auto issue = [&](int kt, const unsigned char *src, unsigned dst, bool v) {
        const int left = kmax - 1 - kt * kKeys;
        src += (int64_t)kt * kKeys * (int64_t)ts2;
        int dr = drow;
        if constexpr (FORM == ROWS_BOTH) asm volatile("" : "+v"(dr));
#pragma unroll
        for (int j = 0; j < PIECES; j++) {
            const int r = dr + j * PK;
            const unsigned c = (unsigned)(dpos ^ (v ? vperm<HD>(r) : kperm<HD>(r))) * 16u;
            ROWS_DMA((unsigned)min(r, left) * ts2 + c, src, dst + j * 1024);
        }
    };
    const unsigned kat = (unsigned)wid * (2 * TILE);
    // (a joint workgroup goes through the prefix and then through its own keys)
    for (int pass = FORM == ROWS_MIXED && p.joint ? 0 : 1; pass < 2; pass++) {
        const bool pre = pass == 0;
        if (FORM == ROWS_MIXED && p.joint) {
            const KeySet &k0 = p.ks[0];
            const int64_t off = (int64_t)kvh * HD;
            ts2 = (unsigned)(pre ? k0.ts : ks.ts) * 2u;
            ksrc = reinterpret_cast<const unsigned char *>(pre ? k0.kv + off : ks.kv + (int64_t)kbatch * ks.bs + off);
            vsrc = ksrc + (int64_t)p.v_off * 2;
            kmax = pre ? (k0.lim ? min(max(k0.lim[kbatch], 0), k0.max_keys) : k0.max_keys) : wmax;
            kt1 = (kmax + kKeys - 1) / kKeys;
        }
        const int plim = pre ? kmax : lim, pmin = pre ? kmax : wmin;
        int kt = wid < NW ? kt0 + wid : kt1;
        bool first = true;
        if (kt < kt1) {
            issue(kt, ksrc, kdst, false);
            issue(kt, vsrc, vdst, true);
        }
        w.wait_q();
        for (; kt < kt1; kt += NW) {
            const bool more = kt + NW < kt1;
            const int kbase = kt * kKeys;
            f32x16 s;
            // (own DMA only, counted in order: K of this tile is behind V of this tile, which is behind K of the next)
            if (PIECES == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
            w.scores(lds, kat, s, [](int) {});
            asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(s) : : "memory");       // the tile's keys have been read
            if (more) issue(kt + NW, ksrc, kdst, false);
            w.softmax(s, kbase + kKeys > pmin, plim - kbase - 4 * h2, first);
            if (!more) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            else if (PIECES == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
            bf16x8_t v[ND];
            w.values(lds, kat + TILE, 0, v);
            w.accumulate(lds, kat + TILE, s, v);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (more) issue(kt + NW, vsrc, vdst, true);
        }
    }
    w.finish();
    __syncthreads();                                           // the tiles are no longer read
    float *sml = reinterpret_cast<float *>(lds + NW * JWAVE);
    if (wid < NW) {
        if (h2 == 0) *reinterpret_cast<float2 *>(sml + (wid * 32 + l32) * 2) = make_float2(w.ms, w.l);
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<float4 *>(lds + wid * JWAVE + l32 * JROW + (32 * d + 2 * e + 4 * h2) * 4) =
                    make_float4(w.o[d][e], w.o[d][e + 1], w.o[d][e + 2], w.o[d][e + 3]);
    }
    __syncthreads();
    // eight threads a row, each every eighth group of four dims; neighbouring threads at neighbouring rows of a partial result's tile, or at
    // neighbouring groups of a row
    const int jr = p.part_o ? tid & 31 : tid >> 3, jq = p.part_o ? tid >> 5 : tid & 7, jt = (row0 + jr) / G, jg = row0 + jr - jt * G;
    if (jt >= n) return;
    float mj[NW], wj[NW], m = kNoKeys, l = 0.0f;
#pragma unroll
    for (int u = 0; u < NW; u++) {
        mj[u] = sml[(u * 32 + jr) * 2];
        m = fmaxf(m, mj[u]);
    }
#pragma unroll
    for (int u = 0; u < NW; u++) {
        wj[u] = __builtin_amdgcn_exp2f(mj[u] - m);
        l += sml[(u * 32 + jr) * 2 + 1] * wj[u];
    }
    const int jtok = n0 + jt, r = jtok * G + jg;
    if (p.part_o && jq == 0) *reinterpret_cast<float2 *>(p.part_ml + ((pt + (r >> 5)) * 32 + (r & 31)) * 2) = make_float2(m, l);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int q = jq; q < HD / 4; q += 8) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < NW; u++) {
            const float4 v = *reinterpret_cast<const float4 *>(lds + u * JWAVE + jr * JROW + q * 16);
            a.x += v.x * wj[u]; a.y += v.y * wj[u]; a.z += v.z * wj[u]; a.w += v.w * wj[u];
        }
        if (p.part_o) *reinterpret_cast<float4 *>(p.part_o + (pt + (r >> 5)) * (32 * HD) + (q * 32 + (r & 31)) * 4) = a;
        else
            *reinterpret_cast<uint2 *>(p.out + (int64_t)jtok * p.o_ts + (int64_t)(kvh * G + jg) * HD + q * 4) =
                make_uint2(f32x2_to_bf16x2(a.x * inv, a.y * inv), f32x2_to_bf16x2(a.z * inv, a.w * inv));
    }
}

// out = sum_j o_j 2^(m_j - m) / sum_j l_j 2^(m_j - m) over the parts j.  Bound by the partial results' bytes where there are many rows
// (12 800 rows of 128 in 5 parts, 33 MB: 7.5 us = 4.4 TB/s), by a few dependent loads otherwise (4 us).  A workgroup takes 32 DG dims of a
// tile of 32 rows: thread (row, q) sums DG groups of four dims (512 bytes in a row for 32 neighbours), eight loads in flight, and works
// out the weights of every eighth part.  The result goes through LDS so that a row's dims are stored in a row.  DG: whole rows where there
// are tiles for the device, else 32 dims.
constexpr int kMaxParts = 128;
template <int HD, int DG>
__global__ __launch_bounds__(256) void k_attn_join(const float *__restrict__ part_o, const float *__restrict__ part_ml, int row_tiles, int nkv,
                                                   int parts, uint16_t *__restrict__ out, int64_t o_ts, int G, int rows,
                                                   const int32_t *__restrict__ cu, int nseqs)
{
    constexpr int U = DG == 1 ? 16 : 8 / DG, KS = 4, OROW = 64 * DG + 16, CH = 4 * DG;
    __shared__ float wts[kMaxParts][32], red[8][32], reds[8][32];
    __shared__ int edges[2];
    __shared__ __attribute__((aligned(16))) unsigned char tile[32 * OROW];
    const int tt = blockIdx.x, d0 = blockIdx.y * 32, kvh = tt / row_tiles, r0 = (tt - kvh * row_tiles) * 32;
    const int tid = threadIdx.x, row = tid & 31, q = tid >> 5;
    const bool ok = r0 + row < rows;
    const int64_t step = (int64_t)nkv * row_tiles;
    const float *po = part_o + (int64_t)tt * (32 * HD) + ((d0 / 4 + q) * 32 + row) * 4;
    float4 v[U][DG];
    auto load = [&](int j, float4 (&x)[DG]) {
#pragma unroll
        for (int g = 0; g < DG; g++)
            x[g] = ok && j < parts ? *reinterpret_cast<const float4 *>(po + j * step * (32 * HD) + g * 1024) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    auto stat = [&](int j) {
        return ok ? *reinterpret_cast<const float2 *>(part_ml + ((j * step + tt) * 32 + row) * 2) : make_float2(kNoKeys, 0.0f);
    };
#pragma unroll
    for (int u = 0; u < U; u++) load(u, v[u]);                 // (on their way while the weights are worked out)
    const int edge = cu && tid < 2 ? cu[tid ? nseqs : 0] : tid ? rows : 0;
    float m = kNoKeys;
    float2 st[KS];                                             // the first 32 parts' stay in registers
#pragma unroll
    for (int k = 0; k < KS; k++) st[k] = q + 8 * k < parts ? stat(q + 8 * k) : make_float2(kNoKeys, 0.0f);
#pragma unroll
    for (int k = 0; k < KS; k++) m = fmaxf(m, st[k].x);
    for (int j = q + 8 * KS; j < parts; j += 8) m = fmaxf(m, stat(j).x);
    red[q][row] = m;
    if (tid < 2) edges[tid] = edge;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; k++) m = fmaxf(m, red[k][row]);
    float l = 0.0f;
    auto weigh = [&](int j, float2 ml) {
        const float w = __builtin_amdgcn_exp2f(ml.x - m);
        wts[j][row] = w;
        l += ml.y * w;
    };
#pragma unroll
    for (int k = 0; k < KS; k++)
        if (q + 8 * k < parts) weigh(q + 8 * k, st[k]);
    for (int j = q + 8 * KS; j < parts; j += 8) weigh(j, stat(j));
    reds[q][row] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) l += reds[k][row];
    float4 a[DG];
#pragma unroll
    for (int g = 0; g < DG; g++) a[g] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < parts; j += U) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (j + u >= parts) break;
            const float w = wts[j + u][row];
#pragma unroll
            for (int g = 0; g < DG; g++) {
                a[g].x += v[u][g].x * w; a[g].y += v[u][g].y * w; a[g].z += v[u][g].z * w; a[g].w += v[u][g].w * w;
            }
            load(j + u + U, v[u]);
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int g = 0; g < DG; g++)
        *reinterpret_cast<uint2 *>(tile + row * OROW + (q + 8 * g) * 8) =
            make_uint2(f32x2_to_bf16x2(a[g].x * inv, a[g].y * inv), f32x2_to_bf16x2(a[g].z * inv, a[g].w * inv));
    __syncthreads();
    for (int i = tid; i < 32 * CH; i += 256) {
        const int rr = i / CH, c = i % CH, r = r0 + rr;
        if (r < rows && r / G >= edges[0] && r / G < edges[1])       // (tokens in front of the first sequence or behind the last: none)
            *reinterpret_cast<uint4 *>(out + (int64_t)(r / G) * o_ts + (int64_t)(kvh * G + r % G) * HD + d0 + c * 8) =
                *reinterpret_cast<const uint4 *>(tile + rr * OROW + c * 16);
    }
}

}  // namespace ifh

using namespace ifh;

extern "C" int ifh_rope_append_packed_bf16(const ifh_rope_packed_desc *d, ifh_stream_t stream)
{
    IFH_CHECK_ARG(d && d->ntokens >= 0 && d->nseqs >= 0);
    if (d->ntokens == 0 || d->nseqs == 0) return IFH_OK;
    IFH_CHECK_ARG(d->qkv && d->q_out && d->cos_sin && d->cache && d->cu && d->pos0 && d->table_len >= 1 && d->max_pos >= 1);
    IFH_CHECK_ARG(d->nheads >= 1 && d->nkv >= 1 && d->head_dim >= 16 && d->head_dim % 16 == 0);
    const int64_t width = (int64_t)(d->nheads + 2 * (int64_t)d->nkv) * d->head_dim;
    IFH_CHECK_ARG(width < (1ll << 24) && d->qkv_ld >= width && d->q_ld >= (int64_t)d->nheads * d->head_dim);
    IFH_CHECK_ARG(d->cache_ts >= (int64_t)2 * d->nkv * d->head_dim && d->cache_bs / d->max_pos >= d->cache_ts);
    IFH_CHECK_ARG(d->qkv_ld % 8 == 0 && d->q_ld % 8 == 0 && d->cache_bs % 8 == 0 && d->cache_ts % 8 == 0);
    IFH_CHECK_ARG(((((uintptr_t)d->qkv) | ((uintptr_t)d->q_out) | ((uintptr_t)d->cache) | ((uintptr_t)d->cos_sin)) & 15) == 0);
    const int64_t total = (int64_t)d->ntokens * (width / 16);
    IFH_CHECK_ARG(total / 256 < (1ll << 31) - 1);
    hipLaunchKernelGGL(k_rope_packed, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, as_stream(stream), (const uint16_t *)d->qkv,
                       d->qkv_ld, (uint16_t *)d->q_out, d->q_ld, d->cos_sin, d->table_len, (uint16_t *)d->cache, d->cache_bs, d->cache_ts,
                       d->cu, d->pos0, d->slot0, d->nseqs, d->nheads, d->nkv, d->head_dim, d->max_pos, total);
    IFH_LAUNCH_CHECK("rope_append_packed");
    return IFH_OK;
}

// Fills in a key set's split for sequences (rows of a batch) of seq_rows rows.
// Narrow workgroups where a narrow block holds a sequence's rows, for packed tokens those of the batch's mean sequence: with more, its keys
// are read once for every 32 rows.  Measured, narrow and wide: 36 rows of 32 sequences behind 1000 keys 15.7 and 16.0 us (with rounded
// probabilities 15.1 and 14.7), 64 rows of 4 behind 4000 14.2 and 14.5 us (13.7 and 13.5); with 6 rows (a decode step of 64 sequences behind
// 1000 keys) 15.6 and 16.7 us.  A batch of long and short sequences has one form for both and is still better off together than in two
// calls: 255 single tokens behind 200-1700 keys and a prompt of 1000, narrow, 65 us, alone 55 and 23; 63 behind 1000-3000 keys and a prompt
// of 512, wide, 50 us, alone 39 and 16.
// A prefix is read by narrow ones as long as seven workgroups for eight CUs do and their rows are four fifths full: its keys then come to
// four waves at once (64 rows of 12 / 2 heads behind 2048 keys 14.9 us, wide 16.3; behind 8000 22.5 and 21.8; 96 rows behind 2048 18.3 and
// 17.3; 8 rows of 40 / 8 heads, 40 rows in two blocks, behind 4000 15.5 and 14.7).
// Keys are split into parts until the device has two workgroups a CU, and no further than that pays for the join's launch and for what
// each part costs it: none of fewer than eight tiles (narrow: two a wave) or four (wide), and at most 1.6 sqrt(tiles) parts, the time of a
// part being tiles / parts and that of the join parts (4 sequences of 4000 keys: 31 parts 15.0 us, 16 parts 13.5 us, 10 parts 14.6 us; one
// of 8000: 63 parts 17.7 us, 25 parts 14.4 us, 15 parts 15.6 us).  Not at all, unless the results are joined anyway, up to 512 keys (wide)
// or 1024 (narrow), and past them while the workgroups that there are (0 to 256) make up for it, wide up to 7 and narrow up to 20 keys a
// workgroup (whole and split: 64 sequences of 16 tokens, 300 keys, 8.7 and 10.4 us; one prompt of 300 rows 10.1 and 11.1 us, of 700 keys 18.8
// and 12.9; 16 of 64 tokens behind 700 keys, 12 / 2 heads, 23.0 and 21.6 us (rounded 19.9 and 20.2), behind 1200 34.4 and 27.4; one token of
// 64 sequences behind 900 keys 15.5 and 19.2 us, behind 2000 30.3 and 36.7; of 16 sequences behind 2000 23.8 and 14.8).
static void split_keys(KeySet *k, bool narrow, int64_t blocks, int nkv, int max_keys)
{
    k->narrow = narrow;
    k->blocks = (int)blocks;
    k->max_keys = max_keys;
    const int tiles = (max_keys + kKeys - 1) / kKeys, least = narrow ? 8 : 4;
    const int64_t want = 2 * (int64_t)device_cu_count_physical() / (blocks * nkv > 0 ? blocks * nkv : 1);
    int parts = (int)(want < 1 ? 1 : want > 64 ? 64 : want);
    if (k->mode == ROWS_PACKED && (tiles <= (narrow ? 32 : 16) || tiles * 32 <= blocks * nkv * (narrow ? 20 : 7))) parts = 1;
    while (2 * (int64_t)parts * parts > 5 * (int64_t)tiles && parts > 1) parts--;
    if (parts > tiles / least) parts = tiles / least > 1 ? tiles / least : 1;
    k->part_tiles = (tiles + parts - 1) / parts;
    k->parts = (tiles + k->part_tiles - 1) / k->part_tiles;
}
static void plan_keys(KeySet *k, int mode, int64_t seq_rows, int64_t blocks_wide, int64_t blocks_narrow, int nkv, int max_keys)
{
    k->mode = mode;
    const bool full = blocks_narrow * kNarrowRows * 4 <= seq_rows * 5;
    if (seq_rows <= kNarrowRows || (mode == ROWS_PREFIX && full)) {
        split_keys(k, true, blocks_narrow, nkv, max_keys);
        if (seq_rows <= kNarrowRows || blocks_narrow * nkv * k->parts * 8 <= 7 * (int64_t)device_cu_count_physical()) return;
    }
    split_keys(k, false, blocks_wide, nkv, max_keys);
}

static int64_t part_floats(int64_t row_tiles, int nkv, int parts, int hd) { return row_tiles * nkv * parts * 32 * (hd + 2); }
static int64_t row_tiles_of(int64_t ntokens, int G) { return (ntokens * G + 31) / 32; }

// one part fewer
static void fewer_parts(KeySet *k)
{
    const int tiles = (k->max_keys + kKeys - 1) / kKeys, parts = k->parts - 1;
    k->part_tiles = (tiles + parts - 1) / parts;
    k->parts = (tiles + k->part_tiles - 1) / k->part_tiles;
}

static void rows_launch(const RowsParams &p, int hd, int form, bool p16, int64_t workgroups, hipStream_t st)
{
    const dim3 grid((unsigned)workgroups), block(256);
#define ROWS_GO(HD, FORM)                                                                         \
    do {                                                                                          \
        if (p16) hipLaunchKernelGGL((k_attn_rows<HD, FORM, true>), grid, block, 0, st, p);        \
        else hipLaunchKernelGGL((k_attn_rows<HD, FORM, false>), grid, block, 0, st, p);           \
    } while (0)
    if (form == ROWS_LONG) {
        if (hd == 128) ROWS_GO(128, ROWS_LONG); else ROWS_GO(64, ROWS_LONG);
    } else if (form == ROWS_BOTH) {
        if (hd == 128) ROWS_GO(128, ROWS_BOTH); else ROWS_GO(64, ROWS_BOTH);
    } else {
        if (hd == 128) ROWS_GO(128, ROWS_MIXED); else ROWS_GO(64, ROWS_MIXED);
    }
#undef ROWS_GO
}

static void join_launch(const RowsParams &p, int hd, int parts, hipStream_t st)
{
    const int tiles = p.row_tiles * p.nkv, rows = p.ntokens * p.G;
    const bool whole = tiles >= device_cu_count_physical();
    const dim3 grid((unsigned)tiles, (unsigned)(whole ? 1 : hd / 32)), block(256);
#define ROWS_JOIN(HD, DG) hipLaunchKernelGGL((k_attn_join<HD, DG>), grid, block, 0, st, p.part_o, p.part_ml, p.row_tiles, p.nkv, parts, p.out, p.o_ts, p.G, rows, p.cu, p.nseqs)
    if (hd == 128) {
        if (whole) ROWS_JOIN(128, 4); else ROWS_JOIN(128, 1);
    } else {
        if (whole) ROWS_JOIN(64, 2); else ROWS_JOIN(64, 1);
    }
#undef ROWS_JOIN
}

static void packed_plan(int64_t ntokens, int64_t nseqs, int G, int nkv, int max_keys, KeySet *k)
{
    plan_keys(k, ROWS_PACKED, (ntokens * G + nseqs - 1) / nseqs, ntokens * G / kWideRows + nseqs, ntokens * G / kNarrowRows + nseqs, nkv, max_keys);
}

// (the callers check that block counts fit an int)
static bool packed_fits(int64_t ntokens, int64_t nseqs, int64_t nheads, int64_t nkv)
{
    return ntokens * (nheads / nkv) < (1ll << 30) && ntokens * nheads < (1ll << 33) && (ntokens * (nheads / nkv) / kNarrowRows + nseqs) * nkv < (1ll << 25);
}

extern "C" int64_t ifh_attn_packed_ws_floats(int ntokens, int nseqs, int nheads, int nkv, int head_dim, int max_keys)
{
    if (ntokens <= 0 || nseqs <= 0 || nkv <= 0 || nheads < nkv || nheads % nkv || max_keys <= 0 || !packed_fits(ntokens, nseqs, nheads, nkv)) return 0;
    KeySet k = {};
    packed_plan(ntokens, nseqs, nheads / nkv, nkv, max_keys, &k);
    return k.parts > 1 ? part_floats(row_tiles_of(ntokens, nheads / nkv), nkv, k.parts, head_dim) : 0;
}

// what the two attention descriptors share
#define IFH_CHECK_HEADS(d)                                                                                                          \
    IFH_CHECK_ARG((d)->nkv >= 1 && (d)->nkv < 65536 && (d)->nheads >= 1 && (d)->nheads <= 65536 && (d)->nheads % (d)->nkv == 0);     \
    IFH_CHECK_ARG((d)->head_dim == 64 || (d)->head_dim == 128);                                                                     \
    IFH_CHECK_ARG((d)->scale > 0.0f && (d)->scale < 1e6f);                                                                          \
    IFH_CHECK_ARG((d)->q_ts >= (int64_t)(d)->nheads * (d)->head_dim && (d)->o_ts >= (int64_t)(d)->nheads * (d)->head_dim);           \
    IFH_CHECK_ARG((d)->v_off >= 0 && (d)->cache_ts >= (int64_t)(d)->v_off + (int64_t)(d)->nkv * (d)->head_dim);                      \
    IFH_CHECK_ARG((d)->cache_ts < (1 << 24) && (d)->cache_bs / (d)->max_keys >= (d)->cache_ts);                                                                  \
    IFH_CHECK_ARG((d)->q_ts % 8 == 0 && (d)->o_ts % 8 == 0 && (d)->cache_bs % 8 == 0 && (d)->cache_ts % 8 == 0 && (d)->v_off % 8 == 0); \
    IFH_CHECK_ARG(((((uintptr_t)(d)->q) | ((uintptr_t)(d)->cache) | ((uintptr_t)(d)->out) | ((uintptr_t)(d)->ws)) & 15) == 0)

extern "C" int ifh_attn_packed_bf16(const ifh_attn_packed_desc *d, ifh_stream_t stream)
{
    IFH_CHECK_ARG(d && d->ntokens >= 0 && d->nseqs >= 0);
    if (d->ntokens == 0 || d->nseqs == 0) return IFH_OK;
    IFH_CHECK_ARG(d->q && d->cache && d->out && d->cu && d->key_len && d->max_keys >= 1 && d->max_keys <= (1 << 30));
    IFH_CHECK_HEADS(d);
    IFH_CHECK_ARG(packed_fits(d->ntokens, d->nseqs, d->nheads, d->nkv));
    RowsParams p = {};
    KeySet &k = p.ks[0];
    p.G = d->nheads / d->nkv;
    packed_plan(d->ntokens, d->nseqs, p.G, d->nkv, d->max_keys, &k);
    k.kv = (const uint16_t *)d->cache; k.bs = d->cache_bs; k.ts = d->cache_ts; k.lim = d->key_len;
    p.q = (const uint16_t *)d->q; p.q_ts = d->q_ts; p.v_off = d->v_off;
    p.out = (uint16_t *)d->out; p.o_ts = d->o_ts;
    p.cu = d->cu;
    p.ntokens = d->ntokens; p.nseqs = d->nseqs; p.nkv = d->nkv; p.T = 1;
    p.scale = d->scale;
    p.row_tiles = (int)row_tiles_of(d->ntokens, p.G);
    while (k.parts > 1 && (!d->ws || part_floats(p.row_tiles, p.nkv, k.parts, d->head_dim) > d->ws_floats)) fewer_parts(&k);
    if (k.parts > 1) {
        p.part_o = d->ws;
        p.part_ml = d->ws + (int64_t)p.row_tiles * p.nkv * k.parts * 32 * d->head_dim;
    }
    const int64_t wgs = (int64_t)k.blocks * p.nkv * k.parts;
    p.first = (int)wgs;
    hipStream_t st = as_stream(stream);
    rows_launch(p, d->head_dim, k.narrow ? ROWS_MIXED : ROWS_LONG, d->probs_bf16, wgs, st);
    IFH_LAUNCH_CHECK("attn_packed");
    if (p.part_o) {
        join_launch(p, d->head_dim, k.parts, st);
        IFH_LAUNCH_CHECK("attn_packed join");
    }
    return IFH_OK;
}

static bool prefix_fits(int64_t ntokens, int64_t nheads, int64_t nkv)
{
    return ntokens < (1 << 24) && ntokens * (nheads / nkv) < (1ll << 30) && (ntokens * (nheads / nkv) / kNarrowRows + ntokens + 1) * nkv < (1ll << 24);
}

// A short prefix is not worth a launch to share it: up to 640 keys in all (five tiles a wave) and two workgroups a CU, the workgroup of a
// row's own keys reads the prefix too (from L2) and writes the result.  Measured, joint and shared: 2 rows of 333 + 40 keys 7.6 and 10.5
// us, 64 rows of 300 + 200 17.3 and 22.3 us (40 / 8 heads); the shared form gains from about 700 keys on (64 rows of 600 + 150 14.4 and
// 11.9 us, 16 rows of 2000 + 200 26.8 and 12.2 us).
static bool prefix_joint(int64_t workgroups, int prefix_keys, int max_keys, bool narrow)
{
    return narrow && (int64_t)prefix_keys + max_keys <= 640 && workgroups <= 2 * (int64_t)device_cu_count_physical();
}

static void prefix_plan(int64_t nrows, int64_t T, int prefix_keys, int nheads, int nkv, int max_keys, KeySet *prefix, KeySet *own)
{
    const int64_t r = T * (nheads / nkv), all = nrows * r;
    plan_keys(prefix, ROWS_PREFIX, all, (all + kWideRows - 1) / kWideRows, (all + kNarrowRows - 1) / kNarrowRows, nkv, prefix_keys);
    plan_keys(own, ROWS_OWN, r, nrows * ((r + kWideRows - 1) / kWideRows), nrows * ((r + kNarrowRows - 1) / kNarrowRows), nkv, max_keys);
}

extern "C" int64_t ifh_attn_prefix_ws_floats(int nrows, int tokens_per_row, int prefix_keys, int nheads, int nkv, int head_dim, int max_keys)
{
    if (nrows <= 0 || tokens_per_row <= 0 || nkv <= 0 || nheads < nkv || nheads % nkv || prefix_keys <= 0 || max_keys <= 0) return 0;
    if (!prefix_fits((int64_t)nrows * tokens_per_row, nheads, nkv)) return 0;
    KeySet a = {}, b = {};
    prefix_plan(nrows, tokens_per_row, prefix_keys, nheads, nkv, max_keys, &a, &b);
    return part_floats(row_tiles_of((int64_t)nrows * tokens_per_row, nheads / nkv), nkv, a.parts + b.parts, head_dim);
}

static int64_t key_workgroups(const KeySet &k, int nkv) { return (int64_t)k.blocks * nkv * k.parts; }
// how many 256s of workgroups of both key sets there are: dealt in turn (ROWS_BOTH) if any
static int prefix_pairs(const KeySet &prefix, const KeySet &own, int nkv)
{
    const int64_t a = key_workgroups(prefix, nkv), b = key_workgroups(own, nkv);
    return (int)((a < b ? a : b) / 256);
}

extern "C" int ifh_attn_prefix_form(int nrows, int tokens_per_row, int prefix_keys, int nheads, int nkv, int max_keys)
{
    if (nrows <= 0 || tokens_per_row <= 0 || nkv <= 0 || nheads < nkv || nheads % nkv || prefix_keys <= 0 || max_keys <= 0) return -1;
    if (!prefix_fits((int64_t)nrows * tokens_per_row, nheads, nkv)) return -1;
    KeySet a = {}, b = {};
    prefix_plan(nrows, tokens_per_row, prefix_keys, nheads, nkv, max_keys, &a, &b);
    const int form = prefix_joint((int64_t)b.blocks * nkv, prefix_keys, max_keys, b.narrow) ? 0 : prefix_pairs(a, b, nkv) > 0 ? 2 : 1;
    return form | a.narrow << 2 | b.narrow << 3;
}

extern "C" int ifh_attn_prefix_bf16(const ifh_attn_prefix_desc *d, ifh_stream_t stream)
{
    IFH_CHECK_ARG(d && d->nrows >= 0);
    if (d->nrows == 0) return IFH_OK;
    IFH_CHECK_ARG(d->q && d->prefix && d->cache && d->out && d->key_len && d->ws && d->tokens_per_row >= 1);
    IFH_CHECK_ARG(d->prefix_keys >= 1 && d->prefix_keys <= (1 << 30) && d->max_keys >= 1 && d->max_keys <= (1 << 30));
    IFH_CHECK_HEADS(d);
    IFH_CHECK_ARG((((uintptr_t)d->prefix) & 15) == 0 && d->prefix_ts % 8 == 0 && d->prefix_ts < (1 << 24) &&
                  d->prefix_ts >= (int64_t)d->v_off + (int64_t)d->nkv * d->head_dim);
    const int64_t ntokens = (int64_t)d->nrows * d->tokens_per_row;
    IFH_CHECK_ARG(prefix_fits(ntokens, d->nheads, d->nkv));
    RowsParams p = {};
    KeySet &a = p.ks[0], &b = p.ks[1];
    prefix_plan(d->nrows, d->tokens_per_row, d->prefix_keys, d->nheads, d->nkv, d->max_keys, &a, &b);
    a.kv = (const uint16_t *)d->prefix; a.ts = d->prefix_ts; a.lim = d->prefix_len;
    b.kv = (const uint16_t *)d->cache; b.bs = d->cache_bs; b.ts = d->cache_ts; b.lim = d->key_len;
    p.q = (const uint16_t *)d->q; p.q_ts = d->q_ts; p.v_off = d->v_off;
    p.out = (uint16_t *)d->out; p.o_ts = d->o_ts;
    p.ntokens = (int)ntokens; p.nseqs = d->nrows; p.nkv = d->nkv; p.G = d->nheads / d->nkv; p.T = d->tokens_per_row;
    p.scale = d->scale;
    p.row_tiles = (int)row_tiles_of(ntokens, p.G);
    while (a.parts + b.parts > 2 && part_floats(p.row_tiles, p.nkv, a.parts + b.parts, d->head_dim) > d->ws_floats) fewer_parts(a.parts >= b.parts ? &a : &b);
    const int parts = a.parts + b.parts;
    b.part0 = a.parts;
    IFH_CHECK_ARG(d->ws_floats >= part_floats(p.row_tiles, p.nkv, parts, d->head_dim));
    hipStream_t st = as_stream(stream);
    if (prefix_joint((int64_t)b.blocks * p.nkv, d->prefix_keys, d->max_keys, b.narrow)) {
        p.joint = 1;
        rows_launch(p, d->head_dim, ROWS_MIXED, d->probs_bf16, (int64_t)b.blocks * p.nkv, st);
        IFH_LAUNCH_CHECK("attn_prefix joint");
        return IFH_OK;
    }
    p.part_o = d->ws;
    p.part_ml = d->ws + (int64_t)p.row_tiles * p.nkv * parts * 32 * d->head_dim;
    const int64_t na = key_workgroups(a, p.nkv), nb = key_workgroups(b, p.nkv);
    p.first = (int)na;
    p.pairs = prefix_pairs(a, b, p.nkv);
    if (p.pairs == 0) {
        // few of either: the own keys' workgroups (more steps each) start first.  64 rows behind 2048 keys, rounded probabilities: 14.8 us, the
        // prefix first 15.9; where both fill the device dealing them in turn, the prefix first, is better (64 rows of 5 tokens behind 8001
        // keys: 110 us, own keys first 117)
        KeySet t = a;
        a = b;
        b = t;
        p.first = (int)nb;
    }
    rows_launch(p, d->head_dim, p.pairs > 0 ? ROWS_BOTH : ROWS_MIXED, d->probs_bf16, na + nb, st);
    IFH_LAUNCH_CHECK("attn_prefix");
    join_launch(p, d->head_dim, parts, st);
    IFH_LAUNCH_CHECK("attn_prefix join");
    return IFH_OK;
}
