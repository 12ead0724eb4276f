// Language-model operators for prompts laid end to end and for decode steps that share a prefix (the serving forms next to llm.hip's
// padded batches; InfernLLMWorker, Cluster/InfernLLMWorker.py:60-119):
//   k_rope_packed    rotary embedding of q and k and the append of k | v to the cache rows, tokens of all sequences end to end.
//   k_attn_rows      softmax(scale q k^T) v of row blocks: a row is one (token, query head), the G heads of a kv head adjacent, so a
//                    K / V tile serves every head of the group and a block of rows covers few tokens (little work past the diagonal).
//   k_attn_join      joins the partial results of row blocks whose keys were split.
#include "common.h"

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

namespace ifh {

// index s of the sequence with cu[s] <= i < cu[s + 1] (cu non-decreasing, n + 1 entries); n where there is none
__device__ __forceinline__ int packed_seq(const int32_t *__restrict__ cu, int n, int i)
{
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid + 1] <= i) lo = mid + 1; else hi = mid;
    }
    return lo < n && cu[lo] <= i ? lo : n;
}

// One thread per (token, head slot, 8 pairs j .. j + 7 of the head): the arithmetic and the roundings of k_rope_append (llm.hip).
__global__ __launch_bounds__(256) void k_rope_packed(const uint16_t *__restrict__ qkv, int64_t qkv_ld, uint16_t *__restrict__ q_out,
                                                     int64_t q_ld, const float *__restrict__ cs, int table_len,
                                                     uint16_t *__restrict__ cache, int64_t cache_bs, int64_t cache_ts,
                                                     const int32_t *__restrict__ cu, const int32_t *__restrict__ pos0,
                                                     const int32_t *__restrict__ slot0, int nseqs, int nh, int nkv, int hd, int max_pos,
                                                     int64_t total)
{
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= total) return;
    const int half = hd >> 1, groups = half >> 3, slots = nh + 2 * nkv;
    const int j = (int)(idx % groups) * 8, slot = (int)((idx / groups) % slots);
    const int64_t i = idx / ((int64_t)groups * slots);
    const int s = packed_seq(cu, nseqs, (int)i);
    if (s >= nseqs) return;
    const int t = (int)i - cu[s], pos = pos0[s] + t, at = (slot0 ? slot0[s] : pos0[s]) + t;
    if (pos < 0 || pos >= table_len) return;
    if (slot >= nh && (at < 0 || at >= max_pos)) return;
    const uint16_t *src = qkv + i * qkv_ld + (int64_t)slot * hd;
    uint16_t *dst = slot < nh ? q_out + i * q_ld + (int64_t)slot * hd
                              : cache + (int64_t)s * cache_bs + (int64_t)at * cache_ts + (int64_t)(slot - nh) * hd;
    const uint4 lo = *reinterpret_cast<const uint4 *>(src + j), hi = *reinterpret_cast<const uint4 *>(src + j + half);
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

// How the rows of a launch find their keys.
//   PACKED   sequence s has the tokens cu[s] .. cu[s+1]-1 and the first key_len[s] keys of cache row s; its last token sees them all,
//            each earlier one a key less (causal, aligned at the end)
//   PREFIX   every token sees the first lim[token / T] keys (all of them without a list) of one shared row
//   OWN      token i of row b = i / T sees the first lim[i] keys of cache row b
enum { ROWS_PACKED, ROWS_PREFIX, ROWS_OWN };

// the keys of a launch's workgroups: `parts` parts of part_tiles tiles for each of `blocks` row blocks and each kv head
struct KeySet {
    const uint16_t *kv;
    int64_t bs, ts;
    const int32_t *lim;
    int max_keys, blocks, parts, part_tiles, part0;      // part0: the first part's place in the partial results
};

struct RowsParams {
    const uint16_t *q;
    int64_t q_ts;
    int v_off;
    uint16_t *out;
    int64_t o_ts;
    const int32_t *cu;
    int ntokens, nseqs, nh, nkv, G, T;
    float scale;
    KeySet ks;
    int64_t part_rows;                     // rows of one part (ntokens * nh)
    float *part_o, *part_ml;               // [parts][part_rows][hd] f32 unnormalised, [parts][part_rows][2] (max, sum); NULL: write out
};

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

// 16 bytes a lane from BASE + VOFF (a lane's offset) to LDS address DST + 16 lane
#define ROWS_DMA(VOFF, BASE, DST)                                                                                          \
    do {                                                                                                                   \
        unsigned keep_;                                                                                                    \
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0" \
                     : "=&s"(keep_) : "v"(VOFF), "s"(BASE), "s"(DST) : "memory");                                          \
    } while (0)

// NW waves of 32 rows each.  S^T = K Q^T and O^T = V^T P^T with the 32 x 32 x 16 MFMA: a lane holds one row's scores of 16 of every 32
// keys, so the softmax of a row is lane-local up to one exchange with lane ^ 32, and P goes from the accumulators of the first product
// into the operand of the second without leaving the lane (its 8 keys are 8 half + {0..3, 8..11} + 4 (lane / 32): V^T is read in that
// order, transposed by ds_read_b64_tr_b16).  P is rounded to bf16 for the second product, as a bf16 model does; sums and maxima are f32.
//
// K / V tiles of 64 keys come by LDS-DMA into two buffers, the next tile in flight while this one is multiplied, one barrier a tile.
// LDS rows are unpadded (the DMA writes 16 bytes a lane in a row), so the 16-byte chunks of key r are permuted on the source side: K chunk
// c at c ^ (r % 16) (head_dim 64: c ^ (r / 2 % 8)), so that the 16 keys a ds_read_b128 reads at once lie in 16 different bank groups;
// V chunks in groups of four, group g at g ^ (r % 4) (head_dim 64: g ^ (r / 2 % 2)), so that the four keys x 64 bytes of a transposed
// read do.
//
// The running maximum is raised only when a tile's exceeds it by more than 2^8 in the exponential (a wave decides at once): p then stays
// below 2^8, sums in f32 lose nothing by it, and the rescaling of the 4 x 16 accumulators is skipped for almost every tile.
template <int HD, int NW, int KT, int MODE>
__global__ __launch_bounds__(NW * 64, 2) void k_attn_rows(const RowsParams p)
{
    constexpr int NS = HD / 16, ND = HD / 32, NC = KT / 32, R = NW * 32, ROWB = HD * 2, TILE = KT * ROWB, BUF = 2 * TILE;
    constexpr int CH = HD / 8, PK = 1024 / ROWB;               // chunks of a key, keys of a DMA instruction
    constexpr int PIECES = TILE / 1024 / NW;                   // DMA instructions a wave issues for K, and for V, of a tile
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * BUF];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, h2 = lane >> 5;
    const KeySet &ks = p.ks;
    // kv head, row block, part: neighbours on different XCDs, so that with 2, 4 or 8 kv heads an XCD's L2 holds its own heads' keys
    const int G = p.G, kvh = blockIdx.x % p.nkv, bp = blockIdx.x / p.nkv, part = bp / ks.blocks;
    int xb = bp - part * ks.blocks;

    // the block's sequence: tokens [n0, n1), first row of the block within it, its cache row and the keys it may read
    int n0, n1, row0, kbatch, klen;
    if (MODE == ROWS_PACKED) {
        // sequence s owns the block slots floor(cu[s] G / R) + s .. : at least ceil(len G / R) of them, so no table of blocks is needed;
        // the last blocks of a long prompt see the most keys and start first.  The lanes probe 64 sequences at a time (one round trip up
        // to 64 sequences, two up to 4096).
        xb = ks.blocks - 1 - xb;
        int lo = 0, range = p.nseqs;
        while (range > 1) {
            const int step = (range + 63) >> 6, at = lo + lane * step;
            const bool le = lane * step < range && (int)((int64_t)p.cu[at] * G / R) + at <= xb;
            const int cnt = __popcll(__ballot(le));
            const int first = (cnt > 0 ? cnt - 1 : 0) * step;
            lo += first;
            range = min(step, range - first);
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        n0 = min(max(p.cu[lo], 0), p.ntokens);
        n1 = min(max(p.cu[lo + 1], n0), p.ntokens);
        const int blk = xb - ((int)((int64_t)n0 * G / R) + lo);
        if (blk < 0 || (int64_t)blk * R >= (int64_t)(n1 - n0) * G) return;
        row0 = blk * R;
        kbatch = lo;
        klen = min(max(ks.lim[lo], 0), ks.max_keys);
    } else if (MODE == ROWS_PREFIX) {
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
    const int n = n1 - n0, row = row0 + wid * 32 + l32, t = row / G, g = row - t * G;
    const bool ok = t < n;
    const int tok = n0 + (ok ? t : 0), head = kvh * G + (ok ? g : 0);
    int lim, wmax, wmin, kmax;                                 // keys this lane's row sees; most and fewest of the wave's rows; most of the block's
    if (MODE == ROWS_PACKED) {
        const int w0 = row0 + wid * 32, past = klen - n + 1;
        lim = ok ? max(past + t, 0) : 0;
        wmax = w0 / G < n ? max(past + min((w0 + 31) / G, n - 1), 0) : 0;
        wmin = max(past + min(w0 / G, n - 1), 0);
        kmax = max(past + min((row0 + R - 1) / G, n - 1), 0);
        wmax = __builtin_amdgcn_readfirstlane(wmax);
        wmin = __builtin_amdgcn_readfirstlane(wmin);
    } else {
        lim = !ok ? 0 : !ks.lim ? klen : min(max(ks.lim[MODE == ROWS_PREFIX ? tok / p.T : tok], 0), klen);
        wmax = lim;
        wmin = ok ? lim : klen;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            wmax = max(wmax, __shfl_xor(wmax, o, 64));
            wmin = min(wmin, __shfl_xor(wmin, o, 64));
        }
        wmax = __builtin_amdgcn_readfirstlane(wmax);
        wmin = __builtin_amdgcn_readfirstlane(wmin);
        kmax = wmax;
        if (NW > 1) {
            int *smax = reinterpret_cast<int *>(lds);
            if (lane == 0) smax[wid] = wmax;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; w++) kmax = max(kmax, smax[w]);
            __syncthreads();
        }
    }
    kmax = __builtin_amdgcn_readfirstlane(kmax);
    int kt0 = 0, kt1 = (kmax + KT - 1) / KT;
    if (p.part_o) {
        kt0 = part * ks.part_tiles;
        kt1 = min(kt1, kt0 + ks.part_tiles);
    }

    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
    float mrun = -1e30f, lrun = 0.0f;
    const float c1 = p.scale * 1.4426950408889634f, raise = 8.0f / c1;

    // DMA: piece j of wave w brings keys (j NW + w) PK .. + PK - 1 of the tile; lane l -> key l / CH of the piece, LDS chunk l % CH
    const unsigned lbase = (unsigned)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)lds);
    const unsigned ts2 = (unsigned)ks.ts * 2u;
    const unsigned char *kbase0 = reinterpret_cast<const unsigned char *>(ks.kv + (int64_t)kbatch * ks.bs + (int64_t)kvh * HD);
    const int64_t voff = (int64_t)p.v_off * 2;
    const int drow = wid * PK + lane / CH, dpos = lane % CH;
    const unsigned kch = (unsigned)(HD == 128 ? dpos ^ (drow & 15) : dpos ^ ((drow >> 1) & 7)) * 16u;
    const unsigned vch = (unsigned)(HD == 128 ? dpos ^ ((drow & 3) << 2) : dpos ^ (((drow >> 1) & 1) << 2)) * 16u;
    auto kchunk = [&](int j) { return kch ^ (unsigned)((HD == 128 ? (j * NW * PK) & 15 : ((j * NW * PK) >> 1) & 7) * 16); };
    auto issue = [&](int kt) {
        const unsigned dst = lbase + (unsigned)(kt & 1) * BUF + (unsigned)wid * 1024u;
        const unsigned char *src = kbase0 + (int64_t)kt * KT * (int64_t)ts2;
        const int left = kmax - 1 - kt * KT;                   // the last key of the block, relative to the tile
        if (left >= KT - 1) {
            const unsigned o0 = (unsigned)drow * ts2;
#pragma unroll
            for (int j = 0; j < PIECES; j++) {
                const unsigned char *sj = src + (int64_t)(j * NW * PK) * (int64_t)ts2;
                ROWS_DMA(o0 + kchunk(j), sj, dst + j * NW * 1024);
                ROWS_DMA(o0 + vch, sj + voff, dst + TILE + j * NW * 1024);
            }
        } else {                                               // past the end: the last key again, masked below
#pragma unroll
            for (int j = 0; j < PIECES; j++) {
                const unsigned o0 = (unsigned)min(drow + j * NW * PK, left) * ts2;
                ROWS_DMA(o0 + kchunk(j), src, dst + j * NW * 1024);
                ROWS_DMA(o0 + vch, src + voff, dst + TILE + j * NW * 1024);
            }
        }
    };
    unsigned ka[NS], va[ND];                                   // LDS offsets of this lane's fragments in buffer 0
#pragma unroll
    for (int d = 0; d < NS; d++) ka[d] = (unsigned)(l32 * ROWB + ((2 * d + h2) ^ (HD == 128 ? l32 & 15 : (l32 >> 1) & 7)) * 16);
    {
        // lane i of a 16-lane group hands in key i / 4, columns 4 (i % 4) .. + 3 of a 4-key x 16-dim block and gets column i
        const int key = 4 * h2 + ((lane & 15) >> 2), c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
        for (int d = 0; d < ND; d++) va[d] = (unsigned)(TILE + key * ROWB + ((4 * d + c) ^ (HD == 128 ? (key & 3) << 2 : ((key >> 1) & 1) << 2)) * 16 + (lane & 1) * 8);
    }

    if (kt0 < kt1) issue(kt0);
    bf16x8_t qf[NS];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p.q + (int64_t)tok * p.q_ts + (int64_t)head * HD + 16 * s + 8 * h2);
        qf[s] = __builtin_bit_cast(bf16x8_t, v);
    }
    // (the loads of q are waited for here, with the first tile: left to hipcc their wait falls behind the next tile's DMA)
#pragma unroll
    for (int s = 0; s < NS; s++) asm volatile("" : : "v"(qf[s]));
    for (int kt = kt0; kt < kt1; kt++) {
        const int kbase = kt * KT;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                                       // the tile has landed, and the other buffer is no longer read
        if (kt + 1 < kt1) issue(kt + 1);
        if (kbase >= wmax) continue;                           // (a wave's rows see nothing of this tile)
        const unsigned char *buf = lds + (kt & 1) * BUF;
        f32x16 s[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) {
            s[c] = (f32x16){0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < NS; d++) {
                const bf16x8_t kf = *reinterpret_cast<const bf16x8_t *>(buf + ka[d] + c * 32 * ROWB);
                s[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[d], s[c], 0, 0, 0);
            }
        }
        // the maxima below are asm (fmaxf on MFMA results costs a canonicalising v_max each), for which hipcc inserts no wait states:
        // 20 here, one more than a 16-pass MFMA's result needs
        if (NC == 2) asm volatile("s_nop 15\n\ts_nop 3" : "+v"(s[0]), "+v"(s[NC - 1]));
        else asm volatile("s_nop 15\n\ts_nop 3" : "+v"(s[0]));
        if (kbase + KT > wmin) {
            const int rel = lim - kbase - 4 * h2;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[c][e] = c * 32 + 8 * (e >> 2) + (e & 3) < rel ? s[c][e] : -INFINITY;
        }
        float mloc = s[0][0];
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 16; e += 2) asm("v_max3_f32 %0, %0, %1, %2" : "+v"(mloc) : "v"(s[c][e]), "v"(s[c][e + 1]));
        mloc = max_half(mloc);
        if (__any(mloc > mrun + raise)) {
            const float mnew = fmaxf(mrun, mloc), alpha = __builtin_amdgcn_exp2f((mrun - mnew) * c1);
            mrun = mnew;
            lrun *= alpha;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= alpha;
        }
        const float ms = mrun * c1;
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                s[c][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][e], c1, -ms));
                ls[e & 3] += s[c][e];
            }
        lrun += (ls[0] + ls[1]) + (ls[2] + ls[3]);
#pragma unroll
        for (int kk = 0; kk < 2 * NC; kk++) {
            const int c = kk >> 1, e0 = (kk & 1) * 8;
            uint4 pb;
            pb.x = f32x2_to_bf16x2(s[c][e0], s[c][e0 + 1]);
            pb.y = f32x2_to_bf16x2(s[c][e0 + 2], s[c][e0 + 3]);
            pb.z = f32x2_to_bf16x2(s[c][e0 + 4], s[c][e0 + 5]);
            pb.w = f32x2_to_bf16x2(s[c][e0 + 6], s[c][e0 + 7]);
            const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, pb);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                typedef __attribute__((address_space(3))) bf16x4_t *lds4;
                const bf16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(buf + va[d] + kk * 16 * ROWB));
                const bf16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(buf + va[d] + (kk * 16 + 8) * ROWB));
                const bf16x8_t vf = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf, o[d], 0, 0, 0);
            }
        }
    }
    lrun += __shfl_xor(lrun, 32, 64);
    const float inv = p.part_o ? 1.0f : lrun > 0.0f ? 1.0f / lrun : 0.0f;
    const int64_t pr = (int64_t)(ks.part0 + part) * p.part_rows + (int64_t)tok * p.nh + head;
    if (p.part_o && ok && h2 == 0) *reinterpret_cast<float2 *>(p.part_ml + pr * 2) = make_float2(mrun, lrun);
    // A lane holds dims 8 i + 4 (lane / 32) .. + 3 of its row: halves of neighbouring groups of eight are exchanged with lane ^ 32, so that
    // a lane stores whole groups (16 bytes of bf16) and a row's two lanes 32 bytes in a row.
    uint16_t *op = p.out + (int64_t)tok * p.o_ts + (int64_t)head * HD;
    float *po = p.part_o + pr * HD;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
            if (p.part_o) {
                if (ok) {
                    *reinterpret_cast<float4 *>(po + 32 * d + 2 * e + 4 * h2) = make_float4(o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]);
                    *reinterpret_cast<float4 *>(po + 32 * d + 2 * e + 8 + 4 * h2) = make_float4(o[d][e + 4], o[d][e + 5], o[d][e + 6], o[d][e + 7]);
                }
            } else {
                typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
                const u32x2 x = __builtin_amdgcn_permlane32_swap(f32x2_to_bf16x2(o[d][e] * inv, o[d][e + 1] * inv),
                                                                 f32x2_to_bf16x2(o[d][e + 4] * inv, o[d][e + 5] * inv), false, false);
                const u32x2 y = __builtin_amdgcn_permlane32_swap(f32x2_to_bf16x2(o[d][e + 2] * inv, o[d][e + 3] * inv),
                                                                 f32x2_to_bf16x2(o[d][e + 6] * inv, o[d][e + 7] * inv), false, false);
                if (ok) *reinterpret_cast<uint4 *>(op + 32 * d + 2 * e + 8 * h2) = make_uint4(x.x, y.x, x.y, y.y);
            }
        }
}

// out = sum_j o_j 2^((m_j - m) c1) / sum_j l_j 2^((m_j - m) c1); a row is HD / 4 lanes.  Lane j of a row reads part j's (max, sum), so
// that the weights cost one round trip; the partial rows come eight at a time.
template <int HD>
__global__ __launch_bounds__(256) void k_attn_join(const float *__restrict__ part_o, const float *__restrict__ part_ml, int64_t rows,
                                                   int parts, float c1, uint16_t *__restrict__ out, int64_t o_ts, int nh)
{
    constexpr int L = HD / 4, U = 8;
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (row >= rows) return;                                   // (whole rows: the exchanges below stay within a row's lanes)
    const int li = threadIdx.x % L, d = li * 4;
    float m = -1e30f;
    for (int j = li; j < parts; j += L) m = fmaxf(m, part_ml[((int64_t)j * rows + row) * 2]);
#pragma unroll
    for (int o = 1; o < L; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, L));
    float l = 0.0f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < parts; j0 += L) {
        float w = 0.0f;
        if (j0 + li < parts) {
            const float2 ml = *reinterpret_cast<const float2 *>(part_ml + ((int64_t)(j0 + li) * rows + row) * 2);
            w = __builtin_amdgcn_exp2f((ml.x - m) * c1);
            l += ml.y * w;
        }
        const int nj = min(L, parts - j0);
        for (int j = 0; j < nj; j += U) {
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                v[u] = *reinterpret_cast<const float4 *>(part_o + ((int64_t)min(j0 + j + u, parts - 1) * rows + row) * HD + d);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float wu = j + u < nj ? __shfl(w, (j + u) & (L - 1), L) : 0.0f;
                a.x += v[u].x * wu; a.y += v[u].y * wu; a.z += v[u].z * wu; a.w += v[u].w * wu;
            }
        }
    }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) l += __shfl_xor(l, o, L);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    uint2 w;
    w.x = f32x2_to_bf16x2(a.x * inv, a.y * inv);
    w.y = f32x2_to_bf16x2(a.z * inv, a.w * inv);
    *reinterpret_cast<uint2 *>(out + (row / nh) * o_ts + (row % nh) * HD + d) = w;
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

// Row blocks are 128 rows (four waves, 64-key tiles) or, where a sequence has no more than about 32 rows, 32 rows (one wave, 32-key tiles
// and 32 KB of LDS, so that five workgroups of a CU keep loads in flight).
struct Tiling {
    int rows, keys, per_cu;
};
static Tiling tiling(int64_t rows_of_a_sequence) { return rows_of_a_sequence <= 40 ? Tiling{32, 32, 5} : Tiling{128, 64, 2}; }

// parts of the keys and tiles per part, for `blocks` workgroups over max_keys keys: enough parts to fill the device, none of fewer than
// min_keys keys
static void split_keys(KeySet *k, const Tiling &t, int64_t workgroups, int min_keys)
{
    const int tiles = (k->max_keys + t.keys - 1) / t.keys, least = min_keys / t.keys;
    const int64_t want = (int64_t)t.per_cu * device_cu_count_physical() / (workgroups > 0 ? workgroups : 1);
    int parts = (int)(want < 1 ? 1 : want > 64 ? 64 : want);
    if (parts > tiles / least) parts = tiles / least > 1 ? tiles / least : 1;
    k->part_tiles = (tiles + parts - 1) / parts;
    k->parts = (tiles + k->part_tiles - 1) / k->part_tiles;
}

static int64_t part_floats(int64_t rows, int parts, int hd) { return rows * parts * (hd + 2); }

template <int MODE>
static void rows_launch(const RowsParams &p, int hd, const Tiling &t, hipStream_t st)
{
    const dim3 grid((unsigned)((int64_t)p.ks.blocks * p.nkv * (p.part_o ? p.ks.parts : 1)));
    if (t.rows == 32) {
        if (hd == 128) hipLaunchKernelGGL((k_attn_rows<128, 1, 32, MODE>), grid, dim3(64), 0, st, p);
        else hipLaunchKernelGGL((k_attn_rows<64, 1, 32, MODE>), grid, dim3(64), 0, st, p);
    } else {
        if (hd == 128) hipLaunchKernelGGL((k_attn_rows<128, 4, 64, MODE>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((k_attn_rows<64, 4, 64, MODE>), grid, dim3(256), 0, st, p);
    }
}

static void join_launch(const RowsParams &p, int hd, int parts, hipStream_t st)
{
    const int64_t rows = p.part_rows, per = 256 / (hd / 4);
    const dim3 grid((unsigned)((rows + per - 1) / per));
    const float c1 = p.scale * 1.4426950408889634f;
    if (hd == 128) hipLaunchKernelGGL(k_attn_join<128>, grid, dim3(256), 0, st, p.part_o, p.part_ml, rows, parts, c1, p.out, p.o_ts, p.nh);
    else hipLaunchKernelGGL(k_attn_join<64>, grid, dim3(256), 0, st, p.part_o, p.part_ml, rows, parts, c1, p.out, p.o_ts, p.nh);
}

// block slots of a packed launch (the rows' sizes are checked by the callers to fit an int)
static int64_t packed_blocks(int64_t ntokens, int64_t nseqs, int G, const Tiling &t) { return ntokens * G / t.rows + nseqs; }

static int64_t packed_plan(int64_t ntokens, int64_t nseqs, int G, int nkv, int max_keys, KeySet *k, Tiling *t)
{
    *t = tiling((ntokens * G + nseqs - 1) / nseqs);
    const int64_t blocks = packed_blocks(ntokens, nseqs, G, *t);
    k->max_keys = max_keys;
    k->blocks = (int)blocks;
    split_keys(k, *t, blocks * nkv, 256);
    return blocks;
}

extern "C" int64_t ifh_attn_packed_ws_floats(int ntokens, int nseqs, int nheads, int nkv, int head_dim, int max_keys)
{
    if (ntokens <= 0 || nseqs <= 0 || nkv <= 0 || nheads < nkv || nheads % nkv || max_keys <= 0) return 0;
    KeySet k = {};
    Tiling t;
    packed_plan(ntokens, nseqs, nheads / nkv, nkv, max_keys, &k, &t);
    return k.parts > 1 ? part_floats((int64_t)ntokens * nheads, k.parts, head_dim) : 0;
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
    const int G = d->nheads / d->nkv;
    IFH_CHECK_ARG((int64_t)d->ntokens * G < (1ll << 30) && (int64_t)d->ntokens * d->nheads < (1ll << 33));
    RowsParams p = {};
    Tiling t;
    const int64_t blocks = packed_plan(d->ntokens, d->nseqs, G, d->nkv, d->max_keys, &p.ks, &t);
    IFH_CHECK_ARG(blocks * d->nkv * p.ks.parts < (1ll << 31));
    p.q = (const uint16_t *)d->q; p.q_ts = d->q_ts; p.v_off = d->v_off;
    p.out = (uint16_t *)d->out; p.o_ts = d->o_ts;
    p.cu = d->cu;
    p.ks.kv = (const uint16_t *)d->cache; p.ks.bs = d->cache_bs; p.ks.ts = d->cache_ts; p.ks.lim = d->key_len;
    p.ntokens = d->ntokens; p.nseqs = d->nseqs; p.nh = d->nheads; p.nkv = d->nkv; p.G = G; p.T = 1;
    p.scale = d->scale;
    p.part_rows = (int64_t)d->ntokens * d->nheads;
    if (d->ws && p.ks.parts > 1) {
        IFH_CHECK_ARG(d->ws_floats >= part_floats(p.part_rows, p.ks.parts, d->head_dim));
        p.part_o = d->ws;
        p.part_ml = d->ws + p.part_rows * p.ks.parts * d->head_dim;
    }
    hipStream_t st = as_stream(stream);
    rows_launch<ROWS_PACKED>(p, d->head_dim, t, st);
    IFH_LAUNCH_CHECK("attn_packed");
    if (p.part_o) {
        join_launch(p, d->head_dim, p.ks.parts, st);
        IFH_LAUNCH_CHECK("attn_packed join");
    }
    return IFH_OK;
}

struct PrefixPlan {
    KeySet prefix, own;
    Tiling pt, ot;
};

static PrefixPlan prefix_plan(int64_t nrows, int64_t T, int prefix_keys, int nheads, int nkv, int max_keys)
{
    PrefixPlan r = {};
    const int64_t G = nheads / nkv;
    r.pt = tiling(nrows * T * G);
    r.ot = tiling(T * G);
    r.prefix.max_keys = prefix_keys;
    r.prefix.blocks = (int)((nrows * T * G + r.pt.rows - 1) / r.pt.rows);
    split_keys(&r.prefix, r.pt, (int64_t)r.prefix.blocks * nkv, 256);
    r.own.max_keys = max_keys;
    r.own.blocks = (int)(nrows * ((T * G + r.ot.rows - 1) / r.ot.rows));
    split_keys(&r.own, r.ot, (int64_t)r.own.blocks * nkv, 256);
    r.own.part0 = r.prefix.parts;
    return r;
}

extern "C" int64_t ifh_attn_prefix_ws_floats(int nrows, int tokens_per_row, int prefix_keys, int nheads, int nkv, int head_dim, int max_keys)
{
    if (nrows <= 0 || tokens_per_row <= 0 || nkv <= 0 || nheads < nkv || nheads % nkv || prefix_keys <= 0 || max_keys <= 0) return 0;
    if ((int64_t)nrows * tokens_per_row * (nheads / nkv) >= (1ll << 30)) return 0;
    const PrefixPlan r = prefix_plan(nrows, tokens_per_row, prefix_keys, nheads, nkv, max_keys);
    return part_floats((int64_t)nrows * tokens_per_row * nheads, r.prefix.parts + r.own.parts, head_dim);
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
    IFH_CHECK_ARG(ntokens < (1 << 24));
    const int G = d->nheads / d->nkv;
    IFH_CHECK_ARG(ntokens * G < (1ll << 30) && ntokens * d->nheads < (1ll << 33));
    const PrefixPlan r = prefix_plan(d->nrows, d->tokens_per_row, d->prefix_keys, d->nheads, d->nkv, d->max_keys);
    IFH_CHECK_ARG((int64_t)r.prefix.blocks * d->nkv * r.prefix.parts < (1ll << 31) && (int64_t)r.own.blocks * d->nkv * r.own.parts < (1ll << 31));
    RowsParams p = {};
    p.q = (const uint16_t *)d->q; p.q_ts = d->q_ts;
    p.v_off = d->v_off;
    p.out = (uint16_t *)d->out; p.o_ts = d->o_ts;
    p.ntokens = (int)ntokens; p.nseqs = d->nrows; p.nh = d->nheads; p.nkv = d->nkv; p.G = G; p.T = d->tokens_per_row;
    p.scale = d->scale;
    p.part_rows = ntokens * d->nheads;
    const int parts = r.prefix.parts + r.own.parts;
    IFH_CHECK_ARG(d->ws_floats >= part_floats(p.part_rows, parts, d->head_dim));
    p.part_o = d->ws;
    p.part_ml = d->ws + p.part_rows * parts * d->head_dim;
    hipStream_t st = as_stream(stream);
    p.ks = r.prefix;
    p.ks.kv = (const uint16_t *)d->prefix; p.ks.ts = d->prefix_ts; p.ks.lim = d->prefix_len;
    rows_launch<ROWS_PREFIX>(p, d->head_dim, r.pt, st);
    IFH_LAUNCH_CHECK("attn_prefix prefix");
    p.ks = r.own;
    p.ks.kv = (const uint16_t *)d->cache; p.ks.bs = d->cache_bs; p.ks.ts = d->cache_ts; p.ks.lim = d->key_len;
    rows_launch<ROWS_OWN>(p, d->head_dim, r.ot, st);
    IFH_LAUNCH_CHECK("attn_prefix own");
    join_launch(p, d->head_dim, parts, st);
    IFH_LAUNCH_CHECK("attn_prefix join");
    return IFH_OK;
}
