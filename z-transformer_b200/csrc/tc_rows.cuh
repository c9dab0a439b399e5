// Attention of rows over the keys that they see -- the last rows of sequences whose keys lie in pages (attention_paged), or
// whole sequences with a window (attention_forward_window) -- on the tensor cores, straight from the f32 keys and values.
//
//     S = q k^T / sqrt(dim),  P = softmax over the seen keys of each row,  out = P v,  lse = max + ln(denominator)
//
// with the arithmetic of tc_fwd16.cuh: every operand is split into two f16 pieces and every product is three MMAs.  What is
// different:
//   rows    A tile's 128 rows are (token, head of the KV group) pairs, token by token: sixteen tokens of eight heads see the
//           same keys, so a short chunk fills a tile, and a window of W keys costs a tile W + 128 / group keys and not W + 128.
//   keys    come as they are.  Converting warps copy a tile's rows into shared memory (cp.async, row by row: each has its
//           page) and write the pieces, scaled by a power of two of the tile's own, as the operand tiles that the MMAs
//           read: in that form nothing is converted before the launch and nothing is kept in memory.  The power of two is the one
//           that the tile before would have had, so that a row is converted as soon as it is there; where it turns out to be off by
//           more than the pieces can bear, or something is not finite, the tile is converted again with care.
//   scales  K's goes into the tile's scores; V's, and the reference maximum of the tile's exponentials, into the factor with
//           which the row threads add the tile's P V to the row: O leaves TMEM after every tile and is summed in registers,
//           with rounding (the tensor core adds with truncation, 2.3e-7 of O for every 64 keys: over a long prefix that is the
//           largest error of all; see kFlushKeyTiles).
//   masks   Which key tiles a CTA visits follows from its first and last position: the sinks' and the window's.  A key that
//           no row of the tile sees is not read and counts as zero.  A value that is not finite does not enter the product,
//           where a weight of zero would not keep it from a row that does not see it: the row threads add it to those that do.
// Roles: two sets of four row warps -- set j & 1 makes P of tile j, each set sums one half of the columns of every tile --,
// four warps that convert K and four that convert V (above 128 columns the same four), a warp that issues S and one that
// issues P V (a thread issues an MMA of N <= 64 every 50 clocks, the pipe takes one every 32), two idle ones that make the
// four a group for setmaxnreg.
// Many rows of a sequence see the same keys: where a launch before this one (rows_planes_kernel) has converted them, whole tiles
// come by bulk copies, and the converting warps' place is taken by row warps, of which some make P and others sum.
// TMEM: Q hi, Q lo (above 128 columns in shared memory), one O buffer (up to 64 columns two), four S/P buffers (of tiles of 128
// keys two): S runs ahead of the rows, so that a set finds the next tile's when it has made P of one and summed those before.
// What bounds it.  Keys converted beforehand: the products.  Four chunks of 512 rows over 8192 keys of 32/8 heads of 128 581 us, 84 % of
// what three f16 products of every seen pair take at the rate of a large bf16 GEMM; a prompt of 16384 with a window of 4096 520 us (86 %).
// A tile's rows need some 19000 clocks besides, one CTA an SM: 13000 until the first product (the query rows' way in 8000 of them), 3500
// for the rows' way out; at T 8192, 32/8 heads, window 1024 that is why the 380 us are 1.6 times their products'.  Keys that
// the CTA converts: the converting warps' instructions and their waits for rows: 32 ragged sequences, window 2048, 16/16 heads of 64,
// 350 us, 3.7 times what their bytes take.
#pragma once

#include "paged_kernels.cuh"
#include "tc_fwd16.cuh"

namespace zt {
namespace tcr {

using namespace tc;
using tcb::block_mult;
using tcb::floats2;
using tcb::fma2;
using tcb::mul2;
using tcf16::max_abs4;
using tcf16::row_max32;
using tcf16::split_q32;
using tcf16::store_q_piece;

constexpr int kConvert = 128;  // threads that convert a tile

template <int TD, bool PLANES>
struct Cfg {
    static constexpr bool kWide = TD > 128;
    // Keys of a tile.  (Narrow heads that convert their own: what a tile costs beside its conversion is shared by twice the keys.  Us,
    // 64 / 128: 32 ragged sequences of 16 heads of 64 378 / 353; converted beforehand, where a tile waits for two S buffers then,
    // batch 4, T 2048, 32/8 heads of 64 206 / 272.)
    static constexpr int BN = kWide ? 32 : (TD == 64 && !PLANES ? 128 : 64);
    static constexpr int OB = TD == 64 ? 2 : 1;     // O buffers
    static constexpr int SB = BN == 128 ? 2 : 4;    // S/P buffers
    static constexpr int KS = (TD == 256 ? 1 : 2) + (PLANES ? 1 : 0), VS = KS;  // slots of K and V tiles
    static constexpr int KP = BN * TD * 2;          // bytes of one piece of a tile
    static constexpr int QL = kWide ? 128 * TD * 2 : 0;
    // What is copied, waited for and converted at a time is 16 keys of a tile (32 of 64 columns): a part.  A thread has CHUNKS 16-byte
    // chunks of it, and a group of converting warps NP parts under way.
    static constexpr int KEYS = TD == 64 ? 32 : 16, PARTS = BN / KEYS, PART = KEYS * TD * 4, CHUNKS = PART / 16 / kConvert;
    static constexpr int GROUPS = PLANES ? 0 : (kWide ? 1 : 2);
    static constexpr int NP = kWide || PLANES ? 4 : 5;
    static constexpr int SETS = PLANES && kWide ? 1 : 2;  // of warps that make P: with tiles of 32 keys of wide heads one keeps up
    static constexpr int kThreads = (PLANES ? 128 * SETS : GROUPS * kConvert) + 256 + 128;
    // registers a thread, of what the launch gives: 640 threads 96 each, 512 threads 128
    static constexpr int kLaunchRegs = kWide ? 128 : 96;
    static constexpr int kRowRegs = kWide ? (PLANES ? 184 : 200) : (PLANES ? 144 : 160);
    static constexpr int kSoftRegs = kWide ? 104 : 80, kConvertRegs = kWide ? 72 : 64, kIssueRegs = kWide ? 40 : 32;
    static constexpr int kShare = 256 * kRowRegs + (PLANES ? 128 * SETS * kSoftRegs : GROUPS * kConvert * kConvertRegs) + 128 * kIssueRegs;
    static_assert(kShare <= kThreads * kLaunchRegs, "the groups share what the launch has");
    static constexpr int cQh = 0, cQl = TD / 2, cO = kWide ? 128 : TD, cS = kWide ? 384 : (OB + 1) * TD;
    static_assert(cO + OB * TD <= cS && cS + SB * BN <= 512, "tensor memory");
    static constexpr int kData = KS * 2 * KP + VS * 2 * KP + GROUPS * NP * PART + QL;
    // The query rows go through shared memory on their way in (kStaged), the finished ones on their way out, where the tiles are, 16
    // bytes apart from a multiple of 128: eight threads' chunks lie in different banks.
    static constexpr int RS = TD * 4 + 16;
    static constexpr bool kStaged = PLANES || !kWide;
    static constexpr int kQ = (PLANES ? kData : (KS + VS) * 2 * KP) - 128 * RS;
    static constexpr int kEarly = 1;  // K tiles that come before the query rows are through
    static_assert(!kStaged || kQ >= 2 * KP, "the query rows are staged where tiles come later");
    static_assert(128 * RS <= kData, "the finished rows are staged where the tiles were");
    static_assert(NP <= 2 * PARTS, "rows are looked up two tiles ahead");
};

struct Shared {
    uint64_t k_full[3], k_free[3], v_full[3], v_free[3], a_ready, s_full[4], p_full[4], pv_done[4], o_full[2], o_free[2];
    uint32_t tmem_base;
    volatile int abort;
    int found;
    RowSpan span;
    float mk[16], mv[16];       // one over the scales of tiles j & 15 (powers of two)
    uint32_t odd[16][4];        // which values' rows of tile j & 15 hold something that is not finite
    alignas(16) uint32_t top[2][2][4];  // [group][unit & 1][warp]: the largest hi piece; or max |x|
    uint32_t seed[2][4];
    float m_ref[8][128];        // the rows' reference maxima of tile j & 7
    float fin_m[2][128], fin_l[2][128], q_top[2][128];
    // elements to the rows of the next tiles' keys (kNone: counts as zero, kNoPage: NaN): of a group's tile j & 3 or, in tiles
    // of 32 keys, of j & 7; and whether some key of the tile is on no page, 32 keys a word
    long long row[1024];
    int holes[8][4];
};
constexpr long long kNone = -1, kNoPage = -2;

struct Params {
    const float *q, *k, *v;  // k, v: the pool's, or [batch, T, width]
    Pages pg;                // (table null: whole sequences of T rows)
    const int *n_keys, *cu_rows;
    int *bad_count;
    float *out, *lse;        // with parts: the parts', out_part and lse_part elements from one to the next
    long long out_part, lse_part;
    int batch, rows, T, n_heads, n_kv_heads, dim, parts;
    Seen seen;
    float scale_log2;
    // Converted beforehand (rows_planes_kernel): every key tile's K hi, K lo, V hi, V lo as shared memory is to hold them, and what
    // Shared holds of the tile; `tiles` of a sequence's KV head.
    uint8_t *planes;
    uint4 *heads;
    int tiles;
};

__device__ __forceinline__ bool rwait(uint64_t *bar, uint32_t parity, Shared *sh) {
    for (uint32_t i = 0; i < (1u << 20); ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255u) == 255u && sh->abort) return false;
    }
    return false;
}
__device__ __forceinline__ void rgive_up(Shared *sh, int code) {
    sh->abort = code;
    atomicMax(&g_tc_status, code);
}
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
                 "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// One over a power of two between 2^-126 and 2^126.
__device__ __forceinline__ float pow2_inverse(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// v -> packed hi pieces and packed lo pieces.  What the hi ones leave of v comes of one instruction each, which takes a half and
// two floats (it is exact: so is the difference).
__device__ __forceinline__ void split(float2 v, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    float2 rest;
    asm("{\n\t.reg .b16 a, b, m;\n\tmov.b32 {a, b}, %2;\n\tmov.b16 m, 0xBC00;\n\t"  // -1
        "fma.rn.f32.f16 %0, a, m, %3;\n\tfma.rn.f32.f16 %1, b, m, %4;\n\t}"
        : "=f"(rest.x), "=f"(rest.y) : "r"(hi), "f"(v.x), "f"(v.y));
    const __half2 l = __floats2half2_rn(rest.x, rest.y);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
// P of sixteen of 32 columns, times kPScale (which rides in the exponent, see tcf16::row_exp32); returns its sum.
__device__ __forceinline__ float row_exp16(const uint32_t (&r)[32], int first, float cs, float off, uint32_t (&ph)[8], uint32_t (&pl)[8]) {
    const float2 cs2 = make_float2(cs, cs), off2 = make_float2(-off, -off);
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const float2 x = fma2(floats2(r[first + i], r[first + i + 1]), cs2, off2);
        const float2 pe = make_float2(ex2(x.x), ex2(x.y));
        sum = tcb::add2(sum, pe);
        split(pe, ph[i >> 1], pl[i >> 1]);
    }
    return sum.x + sum.y;
}

// -inf for those of 32 keys from key0 on that the query at `pos` does not see.
__device__ __forceinline__ void mask_scores(uint32_t (&r)[32], const Seen &v, int key0, int pos) {
    const auto below = [](int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); };  // the first n bits
    uint32_t seen = below(pos - key0 + 1);
    if (v.window > 0) seen &= ~below(pos - v.window - key0 + 1) | below(v.sinks - key0);
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (!(seen >> i & 1u)) r[i] = 0xff800000u;
}

// The key tiles that the rows at positions [first, last] visit, numbered through: those with sinks, then the window's.
struct Tiles {
    int n, sink_tiles, skip;
    __device__ __forceinline__ Tiles(const Seen &s, int first, int last, int BN) {
        const int end = last / BN + 1;
        const int low = s.window > 0 && first >= s.window ? (first - s.window + 1) / BN : 0;
        const int sinks = s.window > 0 ? (int)(((long long)s.sinks + BN - 1) / BN) : 0;
        sink_tiles = sinks < low ? sinks : low;
        skip = low - sink_tiles, n = end - skip;
    }
    __device__ __forceinline__ int at(int j) const { return j < sink_tiles ? j : j + skip; }
};

// The rows of a tile: flat rows [f0, f0 + 128) of a sequence's (token, head of the group) pairs.
struct RowTile {
    int b, begin, count, pos;  // sequence; its first row in q, its rows, the first one's position
    int computed;              // so many of its rows; the rest are NaN
    int f0;
};

template <int TD, bool PAGED, bool PLANES>
__global__ void __launch_bounds__(Cfg<TD, PLANES>::kThreads, 1) attn_rows_tc(const Params p) {
    using C = Cfg<TD, PLANES>;
    constexpr int BN = C::BN, KP = C::KP, KS = C::KS, VS = C::VS, OB = C::OB, SB = C::SB, kThreads = C::kThreads, kIssuer = kThreads / 32 - 4;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *sK = smem, *sV = sK + KS * 2 * KP, *sRaw = sV + VS * 2 * KP, *sQl = sRaw + C::GROUPS * C::NP * C::PART;
    Shared *sh = reinterpret_cast<Shared *>(sQl + C::QL);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = p.n_heads / p.n_kv_heads;
    const int g = blockIdx.y, part = blockIdx.z;
    const int slot = (int)(gridDim.x - 1 - blockIdx.x);  // (of whole sequences the late tiles, which see the most, start first)

    pdl_wait();
    RowTile t{};
    if (PAGED) {
        if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && warp == kIssuer + 3) {
            int bad = 0;
            for (int i = lane; i < p.batch; i += 32) bad += new_rows(p.cu_rows, p.n_keys, i, p.rows, p.pg, true).bad;
            bad = __reduce_add_sync(0xffffffffu, bad);
            if (lane == 0) *p.bad_count = bad;
        }
        // Sequence b has the tiles from first_row_tile(cu_rows[b]) on: as many as it needs, or one more.
        if (threadIdx.x == 0) sh->found = -1;
        __syncthreads();
        bool ascend = true;
        for (int i = threadIdx.x; i < p.batch; i += kThreads) {
            const int lo = row_bound(p.cu_rows, p.rows, i), hi = row_bound(p.cu_rows, p.rows, i + 1);
            ascend &= lo <= hi;
            if (first_row_tile(lo, group, i) <= slot && slot < first_row_tile(hi, group, i + 1)) atomicMax(&sh->found, i);
        }
        ascend = __syncthreads_and(ascend);
        if (threadIdx.x == 0) {  // (one thread, into shared memory: what the others hold of it costs no registers)
            const int b = sh->found;
            if (!ascend) sh->span = row_span(p.cu_rows, p.batch, p.rows, group, slot);
            else if (b < 0) sh->span.b = b;
            else sh->span = RowSpan{b, row_bound(p.cu_rows, p.rows, b), row_bound(p.cu_rows, p.rows, b + 1), p.rows};
        }
        __syncthreads();
        const RowSpan span = sh->span;
        t.b = span.b;
        if (t.b < 0) return;
        const NewRows r = new_rows(p.cu_rows, p.n_keys, t.b, p.rows, p.pg, true);
        t.begin = span.begin, t.count = span.end - span.begin, t.pos = r.pos + (span.begin - r.begin);
        t.computed = r.bad || span.upto < span.begin ? 0 : (span.upto < span.end ? span.upto : span.end) - span.begin;
        t.f0 = (int)(slot - first_row_tile(span.begin, group, t.b)) * 128;
    } else {
        const int per = (int)(((long long)p.T * group + 127) / 128);
        t.b = slot / per, t.begin = t.b * p.T, t.count = t.computed = p.T, t.f0 = (slot - t.b * per) * 128;
    }
    const long long flat = (long long)t.count * group;
    if (t.f0 >= flat) return;
    const auto of_tile = [&](long long end) { return end - t.f0 < 128 ? (int)(end - t.f0) : 128; };
    const int n_rows = of_tile((long long)t.computed * group);
    // a row's place in q, out and lse
    const auto row_head = [&](int r) -> long long {
        const int f = t.f0 + r, i = f / group;
        return (long long)(t.begin + i) * p.n_heads + g * group + (f - i * group);
    };
    if (PAGED && t.computed < t.count) {
        const float nan = __int_as_float(0x7fc00000);
        const int nan0 = n_rows < 0 ? 0 : n_rows, nan1 = of_tile(flat);
        for (int i = nan0 * p.dim + threadIdx.x; i < nan1 * p.dim; i += kThreads) {
            const int r = i / p.dim;
            p.out[part * p.out_part + row_head(r) * p.dim + (i - r * p.dim)] = nan;
        }
        if (p.lse && (int)threadIdx.x >= nan0 && (int)threadIdx.x < nan1) p.lse[part * p.lse_part + row_head(threadIdx.x)] = nan;
        if (n_rows <= 0) return;
    }
    const int pos_first = t.pos + t.f0 / group, pos_last = t.pos + (t.f0 + n_rows - 1) / group;
    const Tiles tiles(p.seen, pos_first, pos_last, BN);
    int n = tiles.n, jb = 0;  // key tiles of this CTA, and the first of them
    if (p.parts > 1) {
        const int per = (n + p.parts - 1) / p.parts;
        jb = part * per;
        n = n - jb < per ? n - jb : per;
        if (n <= 0) {
            if (threadIdx.x < n_rows) p.lse[part * p.lse_part + row_head(threadIdx.x)] = -INFINITY;
            return;
        }
    }
    const auto key0 = [&](int j) { return tiles.at(jb + j) * BN; };

    if (threadIdx.x == 0) {
        for (int i = 0; i < 3; ++i) {
            mbar_init(&sh->k_full[i], 1), mbar_init(&sh->k_free[i], 1);
            mbar_init(&sh->v_full[i], 1), mbar_init(&sh->v_free[i], 1);
        }
        for (int i = 0; i < SB; ++i) mbar_init(&sh->s_full[i], 1), mbar_init(&sh->p_full[i], 4), mbar_init(&sh->pv_done[i], 1);
        for (int i = 0; i < OB; ++i) mbar_init(&sh->o_full[i], 1), mbar_init(&sh->o_free[i], 8);
        mbar_init(&sh->a_ready, 8);
        sh->abort = (smem_u32(smem) & 1023u) ? 100 : 0;
        if (sh->abort) atomicMax(&g_tc_status, 100);
        mbar_fence_init();
    }
    if (warp == kIssuer) tmem_alloc(&sh->tmem_base, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    const int steps = head_steps(p.dim);

    if (warp >= kIssuer) {
        fewer_registers<C::kIssueRegs>();
        if (warp == kIssuer) {
            // -------------------------------------------------------------- S(j) = Q K^T into buffer j % SB
            if (elect_one()) {
                constexpr uint32_t id_s = idesc_f16(128, BN, false, false);
                bool ok = rwait(&sh->a_ready, 0, sh);
                if (!ok) rgive_up(sh, 101);
                const uint32_t k_u32 = smem_u32(sK), ql_u32 = smem_u32(sQl);
                for (int j = 0; ok && j < n; ++j) {
                    const int s = j % KS;
                    // (over P(j - SB), which its product has read)
                    if (!rwait(&sh->k_full[s], (uint32_t)((j / KS) & 1), sh) ||
                        (j >= SB && !rwait(&sh->pv_done[j % SB], (uint32_t)((j / SB - 1) & 1), sh))) { rgive_up(sh, 102); break; }
                    tc_fence_after();
                    const uint32_t cS = C::cS + (j % SB) * BN;
                    const uint64_t bkh = desc_kmajor(k_u32 + (uint32_t)(s * 2 * KP)), bkl = desc_kmajor(k_u32 + (uint32_t)(s * 2 * KP + KP));
                    const uint64_t bql = desc_kmajor(ql_u32);
                    // (the two small terms of the whole contraction first, while there is little to truncate.  The backward forms S in the same
                    // order: where a softmax is saturated, what its dP and delta leave of each other is as good as the two S agree.  64 columns
                    // at a time / at once: out's error at T 8192, window 1024, heads of 128 5.5e-7 / 3.6e-7, at T 1024, window 256, heads of 256
                    // 9.8e-7 / 4.8e-7; a prompt of 16384, window 4096, heads of 128 538 / 524 us.)
#pragma unroll
                    for (int kk = 0; kk < TD / 16; ++kk) {
                        if (kk >= steps) break;
                        const uint32_t bo = (uint32_t)((kk >> 2) * (BN * 128) + (kk & 3) * 32);
                        mma_ts_f16(tmem + cS, tmem + C::cQh + kk * 8, desc_advance(bkl, bo), id_s, kk > 0);
                        if (C::kWide) mma_ss_f16(tmem + cS, desc_advance(bql, (uint32_t)((kk >> 2) * (128 * 128) + (kk & 3) * 32)), desc_advance(bkh, bo), id_s, 1);
                        else mma_ts_f16(tmem + cS, tmem + C::cQl + kk * 8, desc_advance(bkh, bo), id_s, 1);
                    }
#pragma unroll
                    for (int kk = 0; kk < TD / 16; ++kk) {
                        if (kk >= steps) break;
                        mma_ts_f16(tmem + cS, tmem + C::cQh + kk * 8, desc_advance(bkh, (uint32_t)((kk >> 2) * (BN * 128) + (kk & 3) * 32)), id_s, 1);
                    }
                    mma_commit(&sh->k_free[s]);
                    mma_commit(&sh->s_full[j % SB]);
                }
            }
            __syncwarp();
        } else if (warp == kIssuer + 1) {
            // -------------------------------------------------------------- O(j) = P(j) V
            if (elect_one()) {
                const uint32_t id_o = idesc_f16(128, 16 * steps, false, true);
                const uint32_t v_u32 = smem_u32(sV);
                for (int j = 0; j < n; ++j) {
                    const int s = j % VS, ob = j % OB;
                    if (!rwait(&sh->p_full[j % SB], (uint32_t)((j / SB) & 1), sh) || !rwait(&sh->v_full[s], (uint32_t)((j / VS) & 1), sh) ||
                        (j >= OB && !rwait(&sh->o_free[ob], (uint32_t)((j / OB - 1) & 1), sh))) { rgive_up(sh, 103); break; }
                    tc_fence_after();
                    const uint32_t vh = v_u32 + (uint32_t)(s * 2 * KP);
                    const uint64_t mvh = desc_mnmajor_16b(vh, BN * 128), mvl = desc_mnmajor_16b(vh + KP, BN * 128);
                    const uint32_t cS = C::cS + (j % SB) * BN, cO = C::cO + ob * TD;
#pragma unroll
                    for (int kk = 0; kk < BN / 16; ++kk) {
                        const uint32_t ac = (uint32_t)(32 * (kk >> 1) + (kk & 1) * 8);
                        const uint64_t dvh = desc_advance(mvh, kk * 2048), dvl = desc_advance(mvl, kk * 2048);
                        // (the two small terms of the whole contraction first, while there is little to truncate)
                        mma_ts_f16(tmem + cO, tmem + cS + ac, dvl, id_o, kk > 0);
                        mma_ts_f16(tmem + cO, tmem + cS + ac + 16, dvh, id_o, 1);
                    }
#pragma unroll
                    for (int kk = 0; kk < BN / 16; ++kk)
                        mma_ts_f16(tmem + cO, tmem + cS + (uint32_t)(32 * (kk >> 1) + (kk & 1) * 8), desc_advance(mvh, kk * 2048), id_o, 1);
                    mma_commit(&sh->v_free[s]);
                    mma_commit(&sh->o_full[ob]);
                    mma_commit(&sh->pv_done[j % SB]);
                }
            }
            __syncwarp();
        } else if (PLANES && warp == kIssuer + 2) {
            // -------------------------------------------------------------- the converted tiles, in the order in which they are asked for
            if (elect_one() && !sh->abort) {
                const long long first = ((long long)t.b * p.n_kv_heads + g) * p.tiles;
                const auto tile_at = [&](int j) { return first + tiles.at(jb + j); };
                int n_k = 0, n_v = 0;  // copied
                bool ok = true;
                uint4 head = p.heads[tile_at(0)];
                const auto copy_v = [&](int j) {
                    const int s = j % VS;
                    if (j >= VS && !rwait(&sh->v_free[s], (uint32_t)((j / VS - 1) & 1), sh)) { rgive_up(sh, 107), ok = false; return; }
                    mbar_arrive_expect_tx(&sh->v_full[s], 2 * KP);
                    bulk_load(sV + s * 2 * KP, p.planes + tile_at(j) * (4 * KP) + 2 * KP, 2 * KP, &sh->v_full[s]);
                    ++n_v;
                };
                for (int j = 0; ok && j < n; ++j) {
                    const int s = j % KS;
                    if (j == C::kEarly && !rwait(&sh->a_ready, 0, sh)) { rgive_up(sh, 107), ok = false; break; }  // (the query rows lie there until then)
                    const uint4 now = head;
                    if (j + 1 < n) head = p.heads[tile_at(j + 1)];
                    if (j >= KS && !rwait(&sh->k_free[s], (uint32_t)((j / KS - 1) & 1), sh)) { rgive_up(sh, 107), ok = false; break; }
                    sh->mk[j & 15] = __uint_as_float(now.x), sh->mv[j & 15] = __uint_as_float(now.y);
                    sh->odd[j & 15][0] = now.z, sh->odd[j & 15][1] = now.w;
                    mbar_arrive_expect_tx(&sh->k_full[s], 2 * KP);
                    bulk_load(sK + s * 2 * KP, p.planes + tile_at(j) * (4 * KP), 2 * KP, &sh->k_full[s]);
                    ++n_k;
                    while (ok && j >= C::kEarly && n_v < j) copy_v(n_v);
                }
                if (ok && n <= C::kEarly && !rwait(&sh->a_ready, 0, sh)) rgive_up(sh, 107), ok = false;
                while (ok && n_v < n) copy_v(n_v);
                if (sh->abort) {
                    // let the copies in flight land before the CTA's shared memory goes away
                    for (int j = (n_k > KS ? n_k - KS : 0); j < n_k; ++j) mbar_wait(&sh->k_full[j % KS], (uint32_t)((j / KS) & 1));
                    for (int j = (n_v > VS ? n_v - VS : 0); j < n_v; ++j) mbar_wait(&sh->v_full[j % VS], (uint32_t)((j / VS) & 1));
                }
            }
            __syncwarp();
        }
    } else if (!PLANES && warp >= 8) {
        // ------------------------------------------------------------------ keys and values: copied, scaled, split.  A group's
        // units are tiles of K, or of V, or of both in the order in which the MMAs ask for them: K0, K1, V0, K2, V1, ...
        fewer_registers<C::kConvertRegs>();
        const int ct = threadIdx.x & (kConvert - 1), cw = warp & 3, gi = (warp - 8) >> 2;
        constexpr int CPR = TD / 4, CH = C::CHUNKS, NP = C::NP, PARTS = C::PARTS;  // (CPR: chunks of a row)
        constexpr float kAim = 0.25f;  // of block_mult's: the largest magnitude in [2^12, 2^13), with room for eight times as much
        const bool both = C::GROUPS == 1;
        const int n_units = both ? 2 * n : n;
        const long long width = PAGED ? p.pg.width : (long long)p.n_kv_heads * p.dim;
        uint8_t *ring = sRaw + gi * (NP * C::PART);
        const auto unit = [&](int u, bool &is_k) {
            is_k = both ? u == 0 || ((u & 1) && u != n_units - 1) : gi == 0;
            return !both ? u : u == 0 ? 0 : (is_k ? (u + 1) >> 1 : (u == n_units - 1 ? n - 1 : (u >> 1) - 1));
        };
        const auto sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(3 + gi) : "memory"); };
        // where the keys of tile j lie; one that no row of this CTA sees counts as zero
        const auto place = [&](int j) { return both ? j & 7 : gi * 4 + (j & 3); };
        const auto rows_of = [&](int j) { return sh->row + place(j) * BN; };
        // (in two steps: the table is asked a tile's conversion before its answer is used)
        int key = 0, page = 0;
        bool wanted = false;
        const auto ask = [&](int j) {
            wanted = false;
            if (ct >= BN || j >= n) return;
            key = key0(j) + ct;
            wanted = key <= pos_last && (p.seen.window == 0 || key > pos_first - p.seen.window || key < p.seen.sinks);
            if (PAGED && wanted) page = p.pg.table[(long long)t.b * p.pg.max_pages + p.pg.page_of(key)];
        };
        const auto look_up = [&](int j) {
            if (ct < BN / 32 && (both || gi == 1)) sh->odd[j & 15][ct] = 0;
            if (ct >= BN || j >= n) return;
            long long at = kNone;
            if (wanted) at = PAGED ? p.pg.row_on(page, key) : ((long long)t.b * p.T + key) * width;
            if (PAGED && wanted && at < 0) at = kNoPage;
            rows_of(j)[ct] = at;
            const bool hole = PAGED && __any_sync(0xffffffffu, at == kNoPage);
            if (lane == 0) sh->holes[place(j)][cw] = hole;
        };
        // Sixteen rows by eight threads each, a thread the chunks (ct & 7) + 8 i of its row: one look-up and one address a row, whole
        // 128-byte lines a row, and sixteen threads write eight bytes each of two rows whose chunks lie in different banks (rows four
        // apart, see the swizzle).
        const int pr = (ct >> 3 & 1) << 2 | (ct >> 4 & 3) | (ct >> 6) << 3, pc = ct & 7;
        constexpr int CPT = TD / 32;                     // chunks that a thread has of a row
        const int my_chunks = (p.dim / 4 - pc + 7) / 8;  // of the head's columns; the rest of the tile's are zeros
        const bool whole = p.dim == TD;
        const float *k_col = p.k + (long long)g * p.dim + pc * 4, *v_col = p.v + (long long)g * p.dim + pc * 4;
        int cu = 0, cq = 0, cs = 0;  // the part that is copied next: unit, part, place in the ring
        const auto copy_part = [&]() {
            if (cu < n_units) {
                bool is_k;
                const int j = unit(cu, is_k);
                const uint32_t dst = smem_u32(ring) + (uint32_t)(cs * C::PART + ct * 16);
                const float *col = is_k ? k_col : v_col;
#pragma unroll
                for (int r = 0; r < C::KEYS; r += 16) {
                    const long long at = rows_of(j)[cq * C::KEYS + r + pr];
                    const float *src = col + (at >= 0 ? at : 0);
                    const uint32_t to = dst + (r / 16) * CPT * (kConvert * 16);
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < CPT; ++i) copy16_async(to + i * (kConvert * 16), src + i * 32, at >= 0);
                    } else {
                        const int have = at >= 0 ? my_chunks : 0;
#pragma unroll
                        for (int i = 0; i < CPT; ++i) copy16_async(to + i * (kConvert * 16), i < have ? src + i * 32 : p.k, i < have);
                    }
                }
                cs = cs + 1 == NP ? 0 : cs + 1;
                if (++cq == PARTS) cq = 0, ++cu;
            }
            copy_async_commit();
        };
        // Where chunk (r, c) has its pieces in the operand tile: 64-column block, row, 16-byte chunk of eight halves with the
        // 128-byte swizzle, its first or second half.
        const auto piece_at = [](int r, int c) { return (c >> 4) * (BN * 128) + r * 128 + ((((c & 15) >> 1) ^ (r & 7)) << 4) + (c & 1) * 8; };
        const uint32_t piece0 = (uint32_t)piece_at(pr, pc);  // (the thread's other chunks: bit 6 for the odd ones, then the next block)
        // A tile once more, from memory: the scale is its own, keys on no page are NaN, values that are not finite are noted and
        // left to the row threads.  Returns the scale.
        const auto with_care = [&](uint8_t *dst, bool is_k, int j, int u) -> float {
            const auto chunk = [&](int f) {
                const long long at = rows_of(j)[f / CPR];
                const int col = f % CPR * 4;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (at >= 0 && col < p.dim) x = *reinterpret_cast<const float4 *>((is_k ? p.k : p.v) + at + (long long)g * p.dim + col);
                if (is_k && at == kNoPage) x.x = __int_as_float(0x7fc00000);
                return x;
            };
            uint32_t top = 0;
#pragma unroll 1
            for (int f = ct; f < BN * CPR; f += kConvert) {
                const float4 x = chunk(f);
                const int r = f / CPR;
                for (const float e : {x.x, x.y, x.z, x.w}) {
                    if (finite(e)) top = max(top, __float_as_uint(e) & 0x7fffffffu);
                    else if (!is_k) atomicOr(&sh->odd[j & 15][r >> 5], 1u << (r & 31));
                }
            }
            top = __reduce_max_sync(0xffffffffu, top);
            sync();  // (everyone has read what `top` held)
            if (lane == 0) sh->top[gi][u & 1][cw] = top;
            sync();
            const uint32_t *tops = sh->top[gi][u & 1];
            const float m = block_mult(max(max(tops[0], tops[1]), max(tops[2], tops[3]))) * kAim;
#pragma unroll 1
            for (int f = ct; f < BN * CPR; f += kConvert) {
                float4 x = chunk(f);
                if (!is_k) x.x = finite(x.x) ? x.x : 0.f, x.y = finite(x.y) ? x.y : 0.f, x.z = finite(x.z) ? x.z : 0.f, x.w = finite(x.w) ? x.w : 0.f;
                uint2 h, l;
                split(make_float2(x.x * m, x.y * m), h.x, l.x);
                split(make_float2(x.z * m, x.w * m), h.y, l.y);
                uint8_t *at = dst + piece_at(f / CPR, f % CPR);
                *reinterpret_cast<uint2 *>(at) = h;
                *reinterpret_cast<uint2 *>(at + KP) = l;
            }
            fence_async_smem();
            sync();
            return m;
        };
        if (ct < 32) sh->holes[ct >> 2][ct & 3] = 0;  // (not every tile has four words)
        sync();
        for (int j = 0; j < 4; ++j) ask(j), look_up(j);
        sync();
#pragma unroll 1
        for (int i = 0; i < NP; ++i) copy_part();
        bool ok = true;
        float m_k = 0.f, m_v = 0.f;  // the next tile's scales; 0: none yet
        int place_now = 0;           // in the ring, of the part that is converted next
#pragma unroll 1
        for (int u = 0; u < n_units; ++u) {
            bool is_k;
            const int j = unit(u, is_k), s = is_k ? j % KS : j % VS, S = is_k ? KS : VS;
            uint8_t *dst = (is_k ? sK : sV) + s * 2 * KP;
            if (C::kStaged && ok && j == (is_k ? C::kEarly : 0) && !__all_sync(0xffffffffu, rwait(&sh->a_ready, 0, sh))) {
                rgive_up(sh, 104);  // (the query rows lie there until then)
                ok = false;
            }
            if (ok && j >= S && !__all_sync(0xffffffffu, rwait(is_k ? &sh->k_free[s] : &sh->v_free[s], (uint32_t)((j / S - 1) & 1), sh))) {
                rgive_up(sh, 104);
                ok = false;  // (on to the barriers that the other warps wait at)
            }
            if (!both || is_k) ask(j + 4);
            float m = is_k ? m_k : m_v;
            uint32_t top = 0;
#pragma unroll 1
            for (int q = 0; q < PARTS; ++q) {
                copy_async_wait<NP - 1>();
                const float4 *raw = reinterpret_cast<const float4 *>(ring + place_now * C::PART) + ct;
                place_now = place_now + 1 == NP ? 0 : place_now + 1;
                float4 x[CH];
#pragma unroll
                for (int i = 0; i < CH; ++i) x[i] = raw[i * kConvert];
                if (m == 0.f) {  // the first tile: by its first keys
                    float most = 0.f;
#pragma unroll
                    for (int i = 0; i < CH; ++i) most = fmaxf(most, max_abs4(x[i]));
                    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
                    if (lane == 0) sh->seed[gi][cw] = bits;
                    sync();
                    const uint32_t *tops = sh->seed[gi];
                    m = block_mult(max(max(tops[0], tops[1]), max(tops[2], tops[3]))) * kAim;
                }
                if (!ok) continue;
                const float2 mm = make_float2(m, m);
                uint8_t *even = dst + q * (C::KEYS * 128) + piece0, *odd = dst + q * (C::KEYS * 128) + (piece0 ^ 64);
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    uint2 h, l;
                    split(mul2(make_float2(x[i].x, x[i].y), mm), h.x, l.x);
                    split(mul2(make_float2(x[i].z, x[i].w), mm), h.y, l.y);
                    top = __vmaxu2(top, __vmaxu2(h.x & 0x7fff7fffu, h.y & 0x7fff7fffu));
                    uint8_t *at = (i & 1 ? odd : even) + (i % CPT >> 1) * (BN * 128) + (i / CPT) * (16 * 128);
                    *reinterpret_cast<uint2 *>(at) = h;
                    *reinterpret_cast<uint2 *>(at + KP) = l;
                }
                copy_part();  // (into the place of the chunks that this thread has just converted)
            }
            fence_async_smem();
            top = max(top & 0xffffu, top >> 16);
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) sh->top[gi][u & 1][cw] = top;
            int hole = 0;
            if (PAGED && is_k)
                for (int i = 0; i < BN / 32; ++i) hole |= sh->holes[place(j)][i];
            sync();
            const uint4 tops = *reinterpret_cast<const uint4 *>(sh->top[gi][u & 1]);
            top = max(max(tops.x, tops.y), max(tops.z, tops.w));
            // The largest hi piece below 2^4, or none, or not finite: with care.  What is taken as it is has the tile's largest at 2^4 at least, so
            // that lo pieces, to the nearest 2^-24, are off by 2^-29 of it at most, and elements down to 2^-7 of it keep their 22 bits.
            const bool care = top < 0x4c00u || top >= 0x7c00u || (is_k && hole);
            if (care) m = with_care(dst, is_k, j, u);
            if (ct == 0) {
                (is_k ? sh->mk : sh->mv)[j & 15] = pow2_inverse(m);
                if (ok) mbar_arrive(is_k ? &sh->k_full[s] : &sh->v_full[s]);
            }
            // the next tile's: with which this one's largest would have been in [2^12, 2^13)
            if (!care) m *= __uint_as_float((uint32_t)(127 + 27 - (int)(top >> 10)) << 23);
            (is_k ? m_k : m_v) = fminf(fmaxf(m, 0x1p-120f), 0x1p120f);
            if (!both || is_k) look_up(j + 4);
        }
        copy_async_wait<0>();
    } else {
        // ------------------------------------------------------------------ rows.  A thread of a set of four warps has a row; of the
        // two sets that sum, half of its columns.
        const int tid = threadIdx.x & 127;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const bool mine = tid < n_rows;
        const int pos = t.pos + (t.f0 + (mine ? tid : n_rows - 1)) / group;  // (rows past the last repeat it, with q zero)
        const long long rh = mine ? row_head(tid) : 0;
        bool ok = true;
        // The row's pieces of q, a half of its columns by each of 256 threads.  (Shared::q_top has the halves' maxima.)
        const auto place_q = [&](int half) {
            float4 x[TD / 8];
            float top = 0.f;
            if (C::kStaged) {
                // a warp fetches its 32 half rows whole lines at a time (each thread its own half row took 10000 clocks)
                constexpr int N = TD / 8;  // chunks of a half row
                uint8_t *staged = smem + C::kQ + half * (TD * 2);
                // (wide heads' by asynchronous copies: a half row on its way would be 128 registers.  2 sequences of T 1024, window 256, 16/4 heads of
                // 256, us: 60 / 55; of 64 columns 195 / 198)
#pragma unroll(C::kWide ? 1 : N)
                for (int i = 0; i < N; ++i) {
                    // (the row's place is known to its own thread; a division each cost 4000 clocks)
                    const int r = (i * 32 + lane) / N, col = half * (TD / 2) + (i * 32 + lane) % N * 4;
                    const long long row = __shfl_sync(0xffffffffu, rh, r);
                    const bool in = (warp & 3) * 32 + r < n_rows && col < p.dim;
                    if (C::kWide) copy16_async(smem_u32(staged + ((warp & 3) * 32 + r) * C::RS + (i * 32 + lane) % N * 16), in ? p.q + row * p.dim + col : p.q, in);
                    else x[i] = in ? *reinterpret_cast<const float4 *>(p.q + row * p.dim + col) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                if (C::kWide) copy_async_commit(), copy_async_wait<0>();
#pragma unroll
                for (int i = 0; !C::kWide && i < N; ++i)
                    *reinterpret_cast<float4 *>(staged + ((warp & 3) * 32 + (i * 32 + lane) / N) * C::RS + (i * 32 + lane) % N * 16) = x[i];
                __syncwarp();
#pragma unroll
                for (int c = 0; c < TD / 8; ++c) x[c] = *reinterpret_cast<const float4 *>(staged + tid * C::RS + c * 16);
            } else {
#pragma unroll
                for (int c = 0; c < TD / 8; ++c) {
                    const int col = half * (TD / 2) + c * 4;
                    x[c] = mine && col < p.dim ? *reinterpret_cast<const float4 *>(p.q + rh * p.dim + col) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
#pragma unroll
            for (int c = 0; c < TD / 8; ++c) top = fmaxf(top, max_abs4(x[c]));
            sh->q_top[half][tid] = top;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float m = block_mult(__float_as_uint(fmaxf(top, sh->q_top[half ^ 1][tid])));
#pragma unroll
            for (int cb = 0; cb < TD / 64; ++cb) {
                uint32_t qh[16], ql[16];
                split_q32([&](int c) { return x[cb * 8 + c]; }, m, qh, ql);
                tmem_st16(tmem + lane_base + C::cQh + half * (TD / 4) + cb * 16, qh);
                if (C::kWide) store_q_piece(sQl, tid, half * (TD / 64) + cb, ql);
                else tmem_st16(tmem + lane_base + C::cQl + half * (TD / 4) + cb * 16, ql);
            }
            tmem_wait_st();
            if (C::kWide || C::kStaged) fence_async_smem();  // (Q lo, and before the bulk copies that land where the rows were)
            tc_fence_before();
            mbar_arrive_warp(&sh->a_ready);
        };
        // positions of this warp's rows: which tiles need a mask
        const int warp_first = __shfl_sync(0xffffffffu, pos, 0), warp_last = __shfl_sync(0xffffffffu, pos, 31);
        float cs0 = 0.f, m_ref = -INFINITY, l = 0.f;
        // P of tile j over S
        const auto make_p = [&](int j) -> bool {
            if (!__all_sync(0xffffffffu, rwait(&sh->s_full[j % SB], (uint32_t)((j / SB) & 1), sh))) {
                rgive_up(sh, 105);
                return false;
            }
            tc_fence_after();
            if (cs0 == 0.f) cs0 = fmaxf(p.scale_log2 / block_mult(__float_as_uint(fmaxf(sh->q_top[0][tid], sh->q_top[1][tid]))), 1.17549435e-38f);
            const int s0 = key0(j);
            const float cs = fmaxf(cs0 * sh->mk[j & 15], 1.17549435e-38f);
            const uint32_t cS = tmem + lane_base + C::cS + (j % SB) * BN;
            const Seen &v = p.seen;
            const bool masked = s0 + BN - 1 > warp_first || (v.window > 0 && s0 <= warp_last - v.window && s0 + BN > v.sinks);
            // 32 columns of S at a time: of a tile of 64 they come out of TMEM a second time for their exponentials, which costs less
            // than the registers to hold them (that sum the rows, or hold half of O beside them)
            constexpr bool kTwice = BN > 32;
            uint32_t r[32];
            const auto scores = [&](int c) {
                tmem_ld32(cS + c, r);
                tmem_wait_ld();
                if (masked) mask_scores(r, v, s0 + c, pos);
            };
            float mt = -INFINITY;
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
                scores(c);
                mt = row_max32(r, mt);
            }
            mt *= cs;  // cs > 0
            if ((mt > m_ref + tcf16::kRescaleThreshold || m_ref == -INFINITY) && mt != -INFINITY) {
                l *= m_ref == -INFINITY ? 0.f : ex2(m_ref - mt);
                m_ref = mt;
            }
            sh->m_ref[j & 7][tid] = m_ref;
            const float off = ((m_ref == -INFINITY) ? 0.f : m_ref) - 7.0f;  // log2 kPScale: l and O are in P's units
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
                if (kTwice) scores(c);
#pragma unroll
                for (int i = 0; i < 32; i += 16) {
                    uint32_t ph[8], pl[8];
                    l += row_exp16(r, i, cs, off, ph, pl);
                    tmem_st8(cS + c + i / 2, ph);
                    tmem_st8(cS + c + 16 + i / 2, pl);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive_warp(&sh->p_full[j % SB]);
            return true;
        };
        // Adds tile j's P V to the thread's half of the row, which is relative to m_o.
        const auto add_tile = [&](int j, int half, float2(&o)[TD / 4], float &m_o) -> bool {
            const int ob = j % OB;
            if (!__all_sync(0xffffffffu, rwait(&sh->o_full[ob], (uint32_t)((j / OB) & 1), sh))) {
                rgive_up(sh, 106);
                return false;
            }
            tc_fence_after();
            // The next product may go over O once it is in registers: its columns are asked for first, the factors formed meanwhile.
            constexpr int COLS = TD / 2 < 64 || !PLANES || C::kWide ? 32 : 64;
            const uint32_t from = tmem + lane_base + C::cO + ob * TD + half * (TD / 2);
            uint32_t r[COLS / 32][32];
            float w = 0.f;
#pragma unroll
            for (int c = 0; c < TD / 2; c += COLS) {
#pragma unroll
                for (int i = 0; i < COLS; i += 32) tmem_ld32(from + c + i, r[i / 32]);
                if (c == 0) {
                    const float mj = sh->m_ref[j & 7][tid];
                    if (__any_sync(0xffffffffu, mj > m_o)) {
                        const float f = mj > m_o ? ex2(m_o - mj) : 1.f;
                        m_o = fmaxf(m_o, mj);
#pragma unroll
                        for (int i = 0; i < TD / 4; ++i) o[i] = mul2(o[i], make_float2(f, f));
                    }
                    // (no key of the tile or before it is seen: P is zero)
                    w = mj == -INFINITY ? 0.f : ex2(mj - m_o) * sh->mv[j & 15];
                }
                tmem_wait_ld();
                if (c + COLS >= TD / 2) {
                    tc_fence_before();
                    mbar_arrive_warp_relaxed(&sh->o_free[ob]);
                }
#pragma unroll
                for (int i = 0; i < COLS; i += 2)
                    o[(c + i) >> 1] = fma2(floats2(r[i / 32][i % 32], r[i / 32][i % 32 + 1]), make_float2(w, w), o[(c + i) >> 1]);
            }
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) any |= sh->odd[j & 15][i];
            if (any) {  // values that are not finite, added to the rows that see them
#pragma unroll 1
                for (int i = 0; i < BN; ++i) {
                    const int key = key0(j) + i;
                    if (!(sh->odd[j & 15][i >> 5] >> (i & 31) & 1u) || !p.seen(key, pos)) continue;
                    const long long at = PAGED ? p.pg.row(t.b, key) : ((long long)t.b * p.T + key) * ((long long)p.n_kv_heads * p.dim);
                    if (at < 0) continue;
#pragma unroll
                    for (int c = 0; c < TD / 4; ++c) {
                        const int col = half * (TD / 2) + 2 * c;
                        if (col >= p.dim) continue;
                        const float2 x = *reinterpret_cast<const float2 *>(p.v + at + (long long)g * p.dim + col);
                        if (!finite(x.x)) o[c].x += x.x;
                        if (!finite(x.y)) o[c].y += x.y;
                    }
                }
                __syncwarp();
            }
            return true;
        };
        // The row leaves: the sets' sums of exponentials together, then every half as one bulk copy.
        const auto publish_sums = [&](int set) { sh->fin_m[set][tid] = m_ref, sh->fin_l[set][tid] = l; };
        const auto send_rows = [&](int half, const float2(&o)[TD / 4], float m_o) {
            const float m0 = sh->fin_m[0][tid], m1 = C::SETS > 1 ? sh->fin_m[1][tid] : -INFINITY, mm = fmaxf(m0, m1);
            // (a part may hold no key that the row sees)
            const float w0 = m0 == -INFINITY ? 0.f : ex2(m0 - mm), w1 = m1 == -INFINITY ? 0.f : ex2(m1 - mm);
            const float sum = w0 * sh->fin_l[0][tid] + (C::SETS > 1 ? w1 * sh->fin_l[1][tid] : 0.f);
            const float f = m_o == -INFINITY ? sum : ex2(m_o - mm) / sum;  // (sum: zero, or NaN)
            const int c0 = half * (TD / 2), cols = p.dim - c0 < TD / 2 ? p.dim - c0 : TD / 2;
            uint8_t *srow = smem + tid * C::RS + c0 * 4;
#pragma unroll
            for (int c = 0; c < TD / 4; c += 2)
                *reinterpret_cast<float4 *>(srow + c * 8) = make_float4(o[c].x * f, o[c].y * f, o[c + 1].x * f, o[c + 1].y * f);
            tcf16::send_row<false>(p.out + part * p.out_part + rh * p.dim + c0, srow, cols, mine);
            if (half == 0 && p.lse && mine) p.lse[part * p.lse_part + rh] = (mm + log2f(sum) - 7.0f) * kLn2;
        };
        const auto sync_rows = [&]() { asm volatile("bar.sync 2, %0;" ::"n"(PLANES ? 128 * C::SETS + 256 : 256) : "memory"); };
        if (PLANES && warp < 4 * C::SETS) {
            (C::kSoftRegs > C::kLaunchRegs ? more_registers<C::kSoftRegs> : fewer_registers<C::kSoftRegs>)();
            const int set = warp >> 2;
            for (int j = set; ok && j < n; j += C::SETS) ok = make_p(j);
            publish_sums(set);
            sync_rows();
        } else {
            more_registers<C::kRowRegs>();
            const int half = (PLANES ? warp - 4 * C::SETS : warp) >> 2;
            place_q(half);
            float2 o[TD / 4];
#pragma unroll
            for (int c = 0; c < TD / 4; ++c) o[c] = make_float2(0.f, 0.f);
            float m_o = -INFINITY;
            int added = 0;
            if (!PLANES)
                for (int j = half; ok && j < n; j += 2) {
                    ok = make_p(j);
                    for (; ok && added < j; ++added) ok = add_tile(added, half, o, m_o);
                }
            for (; ok && added < n; ++added) ok = add_tile(added, half, o, m_o);
            if (!PLANES) publish_sums(half);
            sync_rows();
            if (ok) send_rows(half, o, m_o);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuer) tmem_dealloc(tmem, 512);
}

// Whether the join reads part i of a row: of the parts that there are those with a weight (one that saw none of the row's keys wrote
// nothing).  A row whose sum is NaN has NaN for every part's weight, so that the weight alone does not say which parts there are.
__host__ __device__ inline bool join_reads(int i, int parts, float weight) { return i < parts && weight != 0.f; }

// out, lse <- the parts'.  A warp per (row, head); a row that belongs to no sequence is left as it is.
__global__ void __launch_bounds__(256) rows_join_kernel(const Params p, float *out, float *lse) {
    pdl_wait();
    pdl_launch();
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= p.lse_part) return;
    const int lane = threadIdx.x & 31, token = (int)(row / p.n_heads), n4 = p.dim >> 2;
    bool from = false, to = false;  // (between the least bound and the greatest)
    for (int b = lane; b <= p.batch; b += 32) from |= p.cu_rows[b] <= token, to |= p.cu_rows[b] > token;
    if (!__any_sync(0xffffffffu, from) || !__any_sync(0xffffffffu, to)) return;
    const float mine = lane < p.parts ? p.lse[lane * p.lse_part + row] : -INFINITY;
    float top = mine;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    float w = (mine == -INFINITY) ? 0.f : ex2((mine - top) * kLog2e), sum = w;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    w = lane < p.parts ? w / sum : 0.f;
    for (int c = lane; c - lane < n4; c += 32) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = 0; i0 < p.parts; i0 += 8) {  // (eight of the parts' chunks under way; beyond the last, a weight of zero)
            float wi[8];
            float4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                wi[i] = __shfl_sync(0xffffffffu, w, i0 + i);
                x[i] = join_reads(i0 + i, p.parts, wi[i]) && c < n4 ? *(reinterpret_cast<const float4 *>(p.out + (i0 + i) * p.out_part + row * p.dim) + c) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                a.x = fmaf(wi[i], x[i].x, a.x), a.y = fmaf(wi[i], x[i].y, a.y), a.z = fmaf(wi[i], x[i].z, a.z), a.w = fmaf(wi[i], x[i].w, a.w);
        }
        if (c < n4) *(reinterpret_cast<float4 *>(out + row * p.dim) + c) = a;
    }
    if (lse && lane == 0) lse[row] = top + log2f(sum) * kLn2;
}

// Key tiles for a launch that reads them converted: a block per (tile, KV head, sequence), half of its threads for K and half for
// V.  Reads f32 rows that some row of the sequence sees, writes as much; bound by memory: four sequences of 8192 keys of 8 heads of 128
// (268 MB in, 268 out) 141 to 150 us, 3.7 TB/s; with two blocks an SM instead of three 181 to 185.
template <int TD, bool PAGED>
__global__ void __launch_bounds__(256, 3) rows_planes_kernel(const Params p) {
    using C = Cfg<TD, true>;
    constexpr int BN = C::BN, KP = C::KP, N = BN / 16 * (TD / 32);  // (N: chunks of a thread)
    __shared__ uint32_t tops[2][4], odd[2];
    pdl_wait();
    pdl_launch();
    const int tile = blockIdx.x, g = blockIdx.y, b = blockIdx.z, key0 = tile * BN;
    int first = 0, last = p.T - 1;  // positions of the sequence's rows
    if (PAGED) {
        const NewRows r = new_rows(p.cu_rows, p.n_keys, b, p.rows, p.pg, true);
        if (r.bad || r.count == 0) return;
        first = r.pos, last = r.pos + r.count - 1;
    }
    // (some row sees it: the first one's window is the lowest)
    const auto seen = [&](int key) { return key <= last && (p.seen.window == 0 || key > first - p.seen.window || key < p.seen.sinks); };
    if (key0 > last || (p.seen.window > 0 && key0 + BN - 1 <= first - p.seen.window && key0 >= p.seen.sinks)) return;  // none of the tile's
    const int ct = threadIdx.x & 127, lane = threadIdx.x & 31;
    const bool is_k = threadIdx.x < 128;
    if (threadIdx.x < 2) odd[threadIdx.x] = 0;
    const int pr = (ct >> 3 & 1) << 2 | (ct >> 4 & 3) | (ct >> 6) << 3, pc = ct & 7;  // (see the converting warps)
    const float *col = (is_k ? p.k : p.v) + (long long)g * p.dim + pc * 4;
    const long long width = PAGED ? p.pg.width : (long long)p.n_kv_heads * p.dim;
    float4 x[N];
    uint32_t holes = 0;
#pragma unroll
    for (int q = 0; q < BN / 16; ++q) {
        const int key = key0 + q * 16 + pr;
        const long long at = !seen(key) ? kNone : PAGED ? p.pg.row(b, key) : ((long long)b * p.T + key) * width;
        if (PAGED && seen(key) && at < 0) holes |= 1u << q;
#pragma unroll
        for (int i = 0; i < TD / 32; ++i)
            x[q * (TD / 32) + i] = at >= 0 && (pc + 8 * i) * 4 < p.dim ? *reinterpret_cast<const float4 *>(col + at + i * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    uint32_t top = 0;
#pragma unroll
    for (int q = 0; q < BN / 16; ++q)
#pragma unroll
        for (int i = 0; i < TD / 32; ++i) {
            float4 &y = x[q * (TD / 32) + i];
            for (float *e : {&y.x, &y.y, &y.z, &y.w}) {
                const bool fine = finite(*e);
                top = max(top, fine ? __float_as_uint(*e) & 0x7fffffffu : 0u);
                if (!fine && !is_k) {
                    *e = 0.f;
                    const int r = q * 16 + pr;
                    atomicOr(&odd[r >> 5], 1u << (r & 31));
                }
            }
            if (PAGED && is_k && (holes >> q & 1u)) y.x = __int_as_float(0x7fc00000);
        }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[is_k ? 0 : 1][(threadIdx.x >> 5) & 3] = top;
    __syncthreads();
    float m[2];
    for (int i = 0; i < 2; ++i) m[i] = block_mult(max(max(tops[i][0], tops[i][1]), max(tops[i][2], tops[i][3]))) * 0.25f;
    const long long at = ((long long)b * p.n_kv_heads + g) * p.tiles + tile;
    if (threadIdx.x == 0) p.heads[at] = make_uint4(__float_as_uint(pow2_inverse(m[0])), __float_as_uint(pow2_inverse(m[1])), odd[0], odd[1]);
    uint8_t *dst = p.planes + at * (4 * KP) + (is_k ? 0 : 2 * KP);
    const float2 mm = is_k ? make_float2(m[0], m[0]) : make_float2(m[1], m[1]);
#pragma unroll
    for (int q = 0; q < BN / 16; ++q)
#pragma unroll
        for (int i = 0; i < TD / 32; ++i) {
            const float4 y = x[q * (TD / 32) + i];
            const int r = q * 16 + pr, c = pc + 8 * i;
            uint2 h, l;
            split(mul2(make_float2(y.x, y.y), mm), h.x, l.x);
            split(mul2(make_float2(y.z, y.w), mm), h.y, l.y);
            uint8_t *to = dst + (c >> 4) * (BN * 128) + r * 128 + ((((c & 15) >> 1) ^ (r & 7)) << 4) + (c & 1) * 8;
            *reinterpret_cast<uint2 *>(to) = h;
            *reinterpret_cast<uint2 *>(to + KP) = l;
        }
}

// Keys of a tile, and bytes of the converted tiles of `keys` keys of `batch` sequences with their heads.
inline int tile_keys(int dim) { return tc_tile_dim(dim) > 128 ? 32 : 64; }
inline long long key_tiles(int keys, int dim) { return ((long long)keys + tile_keys(dim) - 1) / tile_keys(dim); }
inline size_t planes_bytes(int batch, int keys, int n_kv_heads, int dim) {
    return (size_t)batch * n_kv_heads * (size_t)key_tiles(keys, dim) * ((size_t)4 * tile_keys(dim) * tc_tile_dim(dim) * 2 + sizeof(uint4)) + 512;
}
// Whether a launch of its own converts the key tiles, each of which so many row tiles visit.  Us, windows of whole sequences, converted
// by the row tiles / beforehand: heads of 64, two visits 17.4 / 16.8, 55.2 / 48.0, three 34.0 / 32.2; of 128, two 24.9 / 27.4, 49.5 / 55.6, three
// 44.3 / 41.0, 71.9 / 70.0; of 192, two 38.6 / 31.3; of 256, two 77 / 44, 40 / 22.  (Wide heads' row warps have no registers to spare
// beside converting warps.)
inline bool converts_beforehand(long long visits, int dim) { return visits >= (dim > 128 ? 1 : dim > 64 ? 3 : 2); }
// The same for new rows over pages, as far as the host knows them -- the sequences have rows / batch each on average --, with the
// bytes that it takes (0: none), and their bound over smaller calls.  Beyond kPlanesMost the rows convert for themselves.
constexpr size_t kPlanesMost = (size_t)2 << 30;
inline size_t paged_planes_bytes(int batch, int rows, int keys, int n_heads, int n_kv_heads, int dim) {
    const size_t bytes = planes_bytes(batch, keys, n_kv_heads, dim);
    return converts_beforehand((long long)rows * (n_heads / n_kv_heads) / 128 / batch, dim) && bytes <= kPlanesMost ? bytes : 0;
}
inline size_t paged_planes_bound(int batch, int rows, int keys, int n_heads, int n_kv_heads, int dim) {
    const int group = n_heads / n_kv_heads;
    long long most = (long long)rows * group / 128;  // sequences of a call that converts beforehand, at most
    while (most > 0 && !converts_beforehand((long long)rows * group / 128 / most, dim)) --most;
    if (most < 1) return 0;
    const size_t bytes = planes_bytes(batch < most ? batch : (int)most, keys, n_kv_heads, dim);
    return bytes < kPlanesMost ? bytes : kPlanesMost;
}
inline void place_planes(Params &p, void *scratch, int keys) {
    p.tiles = (int)key_tiles(keys, p.dim);
    uint8_t *c = static_cast<uint8_t *>(scratch);
    c += (256 - (reinterpret_cast<uintptr_t>(c) & 255u)) & 255u;
    p.planes = c;
    p.heads = reinterpret_cast<uint4 *>(c + (size_t)p.batch * p.n_kv_heads * p.tiles * ((size_t)4 * tile_keys(p.dim) * tc_tile_dim(p.dim) * 2));
}

// The register shares are taken from what the kernel was compiled to be launched with: less than their sum, and a group that asks
// for its share would wait for good.
template <int TD, bool PAGED, bool PLANES>
inline bool registers_suffice() {
    cudaFuncAttributes a{};
    if (cudaFuncGetAttributes(&a, attn_rows_tc<TD, PAGED, PLANES>) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return a.numRegs * Cfg<TD, PLANES>::kThreads >= Cfg<TD, PLANES>::kShare;
}
template <int TD, bool PAGED, bool PLANES>
inline int launch_as(const Params &p, long long slots, cudaStream_t stream) {
    static const bool suffice = registers_suffice<TD, PAGED, PLANES>();
    if (!suffice) return refuse("attn_rows_tc was not compiled for the registers that its warps share out.");
    const size_t smem = (size_t)Cfg<TD, PLANES>::kData + sizeof(Shared);
    if (optin_smem((const void *)attn_rows_tc<TD, PAGED, PLANES>, smem)) return 1;
    if (PLANES && launch_pdl("rows_planes_kernel", rows_planes_kernel<TD, PAGED>, dim3((unsigned)p.tiles, (unsigned)p.n_kv_heads, (unsigned)p.batch),
                             dim3(256), 0, stream, p))
        return 1;
    const dim3 grid((unsigned)slots, (unsigned)p.n_kv_heads, (unsigned)p.parts);
    return launch_after("attn_rows_tc", attn_rows_tc<TD, PAGED, PLANES>, grid, dim3(Cfg<TD, PLANES>::kThreads), smem, stream, 1, p);
}
template <int TD>
inline int launch_td(const Params &p, long long slots, cudaStream_t stream) {
    if (p.planes) return p.pg.table ? launch_as<TD, true, true>(p, slots, stream) : launch_as<TD, false, true>(p, slots, stream);
    return p.pg.table ? launch_as<TD, true, false>(p, slots, stream) : launch_as<TD, false, false>(p, slots, stream);
}
inline int launch(const Params &p, long long slots, cudaStream_t stream) {
    g_last_path = "tcgen05";
    switch (tc_tile_dim(p.dim)) {
        case 64: return launch_td<64>(p, slots, stream);
        case 128: return launch_td<128>(p, slots, stream);
        case 192: return launch_td<192>(p, slots, stream);
        default: return launch_td<256>(p, slots, stream);
    }
}

inline int launch_join(const Params &p, float *out, float *lse, cudaStream_t stream) {
    return launch_pdl("rows_join_kernel", rows_join_kernel, dim3((unsigned)((p.lse_part + 7) / 8)), dim3(256), 0, stream, p, out, lse);
}

// Row tiles, at most, of `rows` new rows of `batch` sequences.
inline long long row_slots(int batch, int rows, int group) { return (long long)rows * group / 128 + batch; }
// How many parts the keys of a row tile are split into, where a CTA an SM is more than there are row tiles: a part keeps a key tile
// of the longest sequence at least.  One sequence, us with the join, parts of 256 / 128 / 64 keys at least: 77 rows, the last of 1000, 32/8
// heads of 128 25.8 / 20.9 / 20.9, 16 of 516 22.1 / 19.0 / 17.2, 30 of 630, 16/4 heads of 256 63 / 43.5 / 36.0; with a tile, and eight
// parts' chunks under way in the join, 19.7, 15.1, 28.5.  Keys converted beforehand, whole / in parts: 500 of 8500, 4/2 heads of 128 138 / 40,
// 200 of 1700, 16/4 of 256 91 / 42, 200 of 4200, 32/8 of 128 99 / 76.
inline int converted_keys(int dim) { return dim > 128 ? Cfg<256, false>::BN : dim > 64 ? Cfg<128, false>::BN : Cfg<64, false>::BN; }
inline int row_parts(int batch, int rows, int max_seen, int n_heads, int n_kv_heads, int dim) {
    const int group = n_heads / n_kv_heads;
    // (sequences share the rows: a tile each, and one more for every 128 rows)
    const long long full = (long long)rows * group, tiles = full / 128 + (full < batch ? full : batch);
    long long n = split_sm_count() / (tiles * n_kv_heads < 1 ? 1 : tiles * n_kv_heads);
    const long long key_tiles = ((long long)max_seen + converted_keys(dim) - 1) / converted_keys(dim);
    if (n > key_tiles) n = key_tiles;
    return n < 2 ? 1 : (n > 32 ? 32 : (int)n);
}
// The most floats of the parts' rows, of a call of at most so many rows: what row_parts splits is at most a CTA's 128 rows an SM.
inline size_t row_parts_bound(int rows, int n_heads, int dim) {
    const size_t by_rows = (size_t)32 * rows * n_heads, by_blocks = (size_t)split_sm_count() * 128;
    return (by_rows < by_blocks ? by_rows : by_blocks) * ((size_t)dim + 1);
}

}  // namespace tcr
}  // namespace zt
